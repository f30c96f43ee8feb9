// The host side of the attention's, the cache store's, the page pool's and the layer operators' calls: argument checks, the
// packing of the C ABI's structs and the call, which in Python took 8 to 12 us of a call whose kernel takes 4.  The modules
// paged_attention.py, kv_cache.py and mx.py hold the interfaces and say what the arguments mean; the kernels stay behind their C ABI, whose functions
// come in as addresses.

#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>

#include <exception>
#include <optional>
#include <string>
#include <utility>

#include "ns_kv_cache.h"
#include "ns_mx.h"
#include "ns_paged_attention.h"

namespace {

struct Refused {
  std::string why;
};

PyObject* g_attention_error = nullptr;   // exception classes, set once by the modules
PyObject* g_store_error = nullptr;
PyObject* g_mx_error = nullptr;

// A tensor argument, borrowed; NULL for None.
const at::Tensor* tensor(PyObject* o, const char* name) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) throw Refused{std::string(name) + " must be a tensor"};
  return &THPVariable_Unpack(o);
}
const at::Tensor& needed(PyObject* o, const char* name) {
  const at::Tensor* t = tensor(o, name);
  if (t == nullptr) throw Refused{std::string(name) + " must be a tensor"};
  return *t;
}
int64_t number(PyObject* o) {   // an int, or anything that stands for one
  PyObject* i = PyNumber_Index(o);
  if (i == nullptr) throw Refused{""};   // Python's own error is set
  const long long v = PyLong_AsLongLong(i);
  Py_DECREF(i);
  if (v == -1 && PyErr_Occurred()) throw Refused{""};
  return v;
}
template <typename F> F function(PyObject* o) { return reinterpret_cast<F>(PyLong_AsVoidPtr(o)); }

std::string shape_of(const at::Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}

void* at_of(const at::Tensor* t) { return t == nullptr ? nullptr : t->data_ptr(); }
int32_t* words(const at::Tensor* t) { return static_cast<int32_t*>(at_of(t)); }

// int32 on the device and contiguous, or made so; `held` keeps what is made.  With a name, of an integer type.
const at::Tensor& int32_on(const at::Tensor& t, at::Device dev, const char* name, at::Tensor& held) {
  if (t.scalar_type() == at::kInt && t.device() == dev && t.is_contiguous()) return t;
  if (name != nullptr && !c10::isIntegralType(t.scalar_type(), false))
    throw Refused{std::string(name) + " must be an integer tensor"};
  held = t.to(dev, at::kInt).contiguous();
  return held;
}

template <typename Body>
PyObject* guarded(PyObject* error, Body body) {
  try {
    return body();
  } catch (const Refused& r) {
    if (!PyErr_Occurred()) PyErr_SetString(error != nullptr ? error : PyExc_RuntimeError, r.why.c_str());
  } catch (...) {   // torch's own, out of memory among them
    if (!PyErr_Occurred()) torch::translate_exception_to_python(std::current_exception());
  }
  return nullptr;
}

// Other Python threads run meanwhile: around what may wait for the device or its queue (copies, allocations, launches).
// Nothing there touches Python's objects.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

bool arguments(Py_ssize_t got, Py_ssize_t want) {
  if (got == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments expected, %zd given", want, got);
  return false;
}

// The library's functions come as addresses (ctypes has them), the stream as its handle.
//
// store(ns_kv_store, ns_kv_last_error, key, value, k_cache, v_cache, block_tables, seq_lens, query_start_loc, query_lens,
//       block_size, query, inv_freq, out, status, stream handle or -1) -> out, or None
// With a handle of -1 the arguments are only checked.
PyObject* store(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments(n, 16)) return nullptr;
  return guarded(g_store_error, [&]() -> PyObject* {
    const at::Tensor &key = needed(a[2], "key"), &value = needed(a[3], "value"), &kc = needed(a[4], "k_cache"),
                     &vc = needed(a[5], "v_cache"), &bt0 = needed(a[6], "block_tables"), &sl0 = needed(a[7], "seq_lens"),
                     &qsl0 = needed(a[8], "query_start_loc"), &ql0 = needed(a[9], "query_lens");
    const int64_t block_size = number(a[10]);
    const at::Tensor *query = tensor(a[11], "query"), *freq = tensor(a[12], "inv_freq"), *out = tensor(a[13], "out"),
                     *status = tensor(a[14], "status");
    const int64_t handle = number(a[15]);
    if (key.dim() != 3 || kc.dim() != 4 || key.sizes() != value.sizes() || kc.sizes() != vc.sizes())
      throw Refused{"key " + shape_of(key) + " and value " + shape_of(value) + " must match, and k_cache " + shape_of(kc) +
                    " and v_cache " + shape_of(vc)};
    const int64_t total = key.size(0), hkv = key.size(1), d = key.size(2);
    if (kc.size(2) != hkv || kc.size(3) != d)
      throw Refused{"the caches' rows " + shape_of(kc) + " are not the keys' " + shape_of(key)};
    if (kc.size(1) != block_size)
      throw Refused{"block_size " + std::to_string(block_size) + " != the cache's " + std::to_string(kc.size(1))};
    const at::ScalarType type = kc.scalar_type();
    const int dtype = type == at::kBFloat16 ? NS_KV_DTYPE_BF16 : type == at::kHalf ? NS_KV_DTYPE_F16
                      : type == at::kFloat ? NS_KV_DTYPE_F32 : -1;
    if (dtype < 0) throw Refused{std::string("unsupported dtype ") + c10::toString(type) + " (float32, bfloat16, float16)"};
    const at::Device dev = kc.device();
    if (query == nullptr) {
      if (out != nullptr) throw Refused{"out is where the rotated query goes: it needs query"};
    } else {
      if (freq == nullptr) throw Refused{"a query is there to be rotated: it needs inv_freq"};
      if (query->dim() != 3 || query->size(0) != total || query->size(2) != d)
        throw Refused{"query " + shape_of(*query) + " does not match the keys' " + shape_of(key)};
    }
    if (freq != nullptr && (freq->scalar_type() != at::kFloat || freq->dim() != 1 || freq->size(0) != d / 2 ||
                            freq->device() != dev || !freq->is_contiguous()))
      throw Refused{"inv_freq must be a contiguous float32 tensor of " + std::to_string(d / 2) +
                    " elements on the cache's device"};
    if (out != nullptr && out->sizes() != query->sizes()) throw Refused{"out must match query's shape"};
    const std::pair<const char*, const at::Tensor*> rows[] = {{"key", &key}, {"value", &value}, {"k_cache", &kc},
                                                              {"v_cache", &vc}, {"query", query}, {"out", out}};
    for (const auto& [name, t] : rows) {
      if (t == nullptr) continue;
      if (t->scalar_type() != type || t->device() != dev)
        throw Refused{std::string(name) + " must share the cache's dtype and device"};
      if (t->stride(-1) != 1) throw Refused{std::string(name) + " must have a unit head_dim stride"};
    }
    if (status != nullptr && (status->scalar_type() != at::kInt || status->device() != dev || status->numel() < 1))
      throw Refused{"status must be an int32 device tensor"};
    if (bt0.dim() != 2) throw Refused{"block_tables must have two dimensions"};
    const int64_t num_seqs = bt0.size(0);
    if (sl0.numel() != num_seqs || ql0.numel() != num_seqs || qsl0.numel() != num_seqs + 1)
      throw Refused{"seq_lens/query_lens need num_seqs entries and query_start_loc num_seqs + 1"};
    if (!dev.is_cuda()) throw Refused{"store_kv_hip needs device tensors"};
    if (handle == -1) Py_RETURN_NONE;
    const auto call = function<decltype(&ns_kv_store)>(a[0]);
    const auto why = function<decltype(&ns_kv_last_error)>(a[1]);
    at::Tensor made, h[4];
    std::optional<Unlocked> meanwhile(std::in_place);
    if (query != nullptr && out == nullptr) {
      made = at::empty_like(*query);
      if (made.stride(-1) != 1) made = at::empty(query->sizes(), query->options());
      out = &made;
    }
    if (total > 0) {
      const bool as_it_is = bt0.scalar_type() == at::kInt && bt0.device() == dev && bt0.stride(1) == 1;
      const at::Tensor& bt = as_it_is ? bt0 : int32_on(bt0, dev, "block_tables", h[0]);
      const at::Tensor &sl = int32_on(sl0, dev, "seq_lens", h[1]), &qsl = int32_on(qsl0, dev, "query_start_loc", h[2]),
                       &ql = int32_on(ql0, dev, "query_lens", h[3]);
      ns_kv_store_args s = {};
      s.query = at_of(query);
      s.key = key.data_ptr();
      s.value = value.data_ptr();
      s.k_cache = kc.data_ptr();
      s.v_cache = vc.data_ptr();
      s.out = query != nullptr ? out->data_ptr() : nullptr;
      s.inv_freq = static_cast<const float*>(at_of(freq));
      s.block_tables = words(&bt);
      s.seq_lens = words(&sl);
      s.query_start_loc = words(&qsl);
      s.query_lens = words(&ql);
      s.status = words(status);
      if (query != nullptr) {
        s.stride_q_token = query->stride(0);
        s.stride_q_head = query->stride(1);
        s.stride_o_token = out->stride(0);
        s.stride_o_head = out->stride(1);
        s.num_heads_q = (int32_t)query->size(1);
      }
      s.stride_key_token = key.stride(0);
      s.stride_key_head = key.stride(1);
      s.stride_value_token = value.stride(0);
      s.stride_value_head = value.stride(1);
      s.stride_k_block = kc.stride(0);
      s.stride_k_token = kc.stride(1);
      s.stride_k_head = kc.stride(2);
      s.stride_v_block = vc.stride(0);
      s.stride_v_token = vc.stride(1);
      s.stride_v_head = vc.stride(2);
      s.stride_bt_seq = bt.stride(0);
      s.total = (int32_t)total;
      s.num_seqs = (int32_t)num_seqs;
      s.num_kv_heads = (int32_t)hkv;
      s.head_dim = (int32_t)d;
      s.block_size = (int32_t)block_size;
      s.num_blocks = (int32_t)kc.size(0);
      s.max_blocks_per_seq = (int32_t)bt.size(1);
      s.dtype = dtype;
      if (call(&s, reinterpret_cast<hipStream_t>(handle)) != 0) throw Refused{why()};
    }
    meanwhile.reset();
    if (query == nullptr) Py_RETURN_NONE;
    if (!made.defined()) {
      Py_INCREF(a[13]);
      return a[13];
    }
    return THPVariable_Wrap(made);
  });
}

// attend(ns_paged_attention_call_workspace, ns_paged_attention, their windowed forms, ns_pa_last_error, query, k_cache,
//        v_cache, block_tables, seq_lens, query_start_loc, query_lens, scale, block_size, max_seq_len, decode_tokens
//        address, their number, prefill_tiles address or 0, their number, window or 0, sinks, out, workspace, counters,
//        status, stream handle or -1) -> out, or the number of counters needed where `counters` is None or the module's
//        own (counters_grow) and too small
// With a handle of -1 the tensors are only checked.
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments(n, 27)) return nullptr;
  return guarded(g_attention_error, [&]() -> PyObject* {
    const at::Tensor &q = needed(a[5], "query"), &kc = needed(a[6], "k_cache"), &vc = needed(a[7], "v_cache"),
                     &bt0 = needed(a[8], "block_tables"), &sl0 = needed(a[9], "seq_lens"),
                     &qsl0 = needed(a[10], "query_start_loc"), &ql0 = needed(a[11], "query_lens");
    const double scale = PyFloat_AsDouble(a[12]);
    if (scale == -1.0 && PyErr_Occurred()) throw Refused{""};
    const int64_t block_size = number(a[13]);
    const at::Tensor *out = tensor(a[21], "out"), *ws = tensor(a[22], "workspace"), *counters = tensor(a[23], "counters"),
                     *status = tensor(a[24], "status");
    const bool counters_grow = PyObject_IsTrue(a[25]) != 0;
    const int64_t handle = number(a[26]);
    if (q.dim() != 3 || kc.dim() != 4) throw Refused{"query must have three dimensions and the caches four"};
    const int64_t total = q.size(0), hq = q.size(1), d = q.size(2);
    const at::ScalarType type = q.scalar_type();
    const at::Device dev = q.device();
    if (kc.sizes() != vc.sizes() || kc.size(3) != d)
      throw Refused{"cache shapes " + shape_of(kc) + ", " + shape_of(vc) + " do not match the query's head_dim " +
                    std::to_string(d)};
    if (kc.scalar_type() != type || vc.scalar_type() != type) throw Refused{"query and caches must share one dtype"};
    if (kc.size(1) != block_size)
      throw Refused{"block_size " + std::to_string(block_size) + " != the cache's " + std::to_string(kc.size(1))};
    if (kc.device() != dev || vc.device() != dev) throw Refused{"query and caches must be on one device"};
    at::Tensor made, held[4];
    auto answer = [&]() -> PyObject* {
      if (made.defined()) return THPVariable_Wrap(made);
      Py_INCREF(a[21]);
      return a[21];
    };
    if (total == 0) {   // nothing to attend (an empty tensor's strides are arbitrary)
      if (out == nullptr) made = at::empty_like(q);
      return answer();
    }
    const std::pair<const char*, const at::Tensor*> rows[] = {{"query", &q}, {"k_cache", &kc}, {"v_cache", &vc}};
    for (const auto& [name, t] : rows)
      if (t->stride(-1) != 1) throw Refused{std::string(name) + " must have a unit head_dim stride"};
    const int64_t num_seqs = bt0.dim() > 0 ? bt0.size(0) : 0;
    if (sl0.numel() != num_seqs || ql0.numel() != num_seqs || qsl0.numel() != num_seqs + 1)
      throw Refused{"seq_lens/query_lens need num_seqs entries and query_start_loc num_seqs + 1"};
    if (out != nullptr && (out->sizes() != q.sizes() || out->scalar_type() != type || out->device() != dev))
      throw Refused{"out must match query's shape, dtype and device"};
    if (out != nullptr && out->stride(-1) != 1) throw Refused{"out must have a unit head_dim stride"};
    if (status != nullptr && (status->scalar_type() != at::kInt || status->device() != dev || status->numel() < 1))
      throw Refused{"status must be an int32 device tensor"};
    const int dtype = type == at::kBFloat16 ? NS_PA_DTYPE_BF16 : type == at::kHalf ? NS_PA_DTYPE_F16
                      : type == at::kFloat ? NS_PA_DTYPE_F32 : -1;
    if (dtype < 0) throw Refused{std::string("unsupported dtype ") + c10::toString(type) + " (float32, bfloat16, float16)"};
    if (handle == -1) Py_RETURN_NONE;
    ns_paged_attn_args s = {};
    s.max_seq_len = (int32_t)number(a[14]);
    s.decode_tokens = reinterpret_cast<const int32_t*>(number(a[15]));
    s.n_decode_tokens = (int32_t)number(a[16]);
    s.prefill_tiles = reinterpret_cast<const int32_t*>(number(a[17]));
    s.n_prefill_tiles = (int32_t)number(a[18]);
    const int64_t window = number(a[19]), sinks = number(a[20]);
    const auto sizes = function<decltype(&ns_paged_attention_call_workspace)>(a[0]);
    const auto call = function<decltype(&ns_paged_attention)>(a[1]);
    const auto window_sizes = function<decltype(&ns_paged_attention_windowed_workspace)>(a[2]);
    const auto window_call = function<decltype(&ns_paged_attention_windowed)>(a[3]);
    const auto why = function<decltype(&ns_pa_last_error)>(a[4]);
    std::optional<Unlocked> meanwhile(std::in_place);
    const at::Tensor &bt = int32_on(bt0, dev, nullptr, held[0]), &sl = int32_on(sl0, dev, nullptr, held[1]),
                     &qsl = int32_on(qsl0, dev, nullptr, held[2]), &ql = int32_on(ql0, dev, nullptr, held[3]);
    if (out == nullptr) {
      made = at::empty_like(q);
      out = &made;
    }
    s.query = q.data_ptr();
    s.k_cache = kc.data_ptr();
    s.v_cache = vc.data_ptr();
    s.out = out->data_ptr();
    s.block_tables = words(&bt);
    s.seq_lens = words(&sl);
    s.query_start_loc = words(&qsl);
    s.query_lens = words(&ql);
    s.status = words(status);
    s.stride_q_token = q.stride(0);
    s.stride_q_head = q.stride(1);
    s.stride_k_block = kc.stride(0);
    s.stride_k_token = kc.stride(1);
    s.stride_k_head = kc.stride(2);
    s.stride_v_block = vc.stride(0);
    s.stride_v_token = vc.stride(1);
    s.stride_v_head = vc.stride(2);
    s.stride_o_token = out->stride(0);
    s.stride_o_head = out->stride(1);
    s.max_blocks_per_seq = bt.dim() == 2 ? (int32_t)bt.size(1) : 0;
    s.stride_bt_seq = s.max_blocks_per_seq;   // contiguous
    s.total_q = (int32_t)total;
    s.num_seqs = (int32_t)num_seqs;
    s.num_heads_q = (int32_t)hq;
    s.num_kv_heads = (int32_t)kc.size(2);
    s.head_dim = (int32_t)d;
    s.block_size = (int32_t)block_size;
    s.num_blocks = (int32_t)kc.size(0);
    s.dtype = dtype;
    s.scale = (float)scale;
    auto checked = [&](int rc) {
      if (rc != 0) throw Refused{why()};
    };
    uint64_t need = 0, count = 0;
    checked(window == 0 ? sizes(&s, &need, &count) : window_sizes(&s, (int32_t)window, (int32_t)sinks, &need, &count));
    at::Tensor room;
    if (need > 0) {
      if (ws != nullptr && (uint64_t)ws->numel() * ws->element_size() < need)
        throw Refused{"workspace of " + std::to_string(need) + " bytes needed, " +
                      std::to_string(ws->numel() * ws->element_size()) + " given (total_q " + std::to_string(total) +
                      ", max_seq_len " + std::to_string(s.max_seq_len) + ", " +
                      std::to_string(s.prefill_tiles != nullptr ? s.n_decode_tokens : s.total_q) + " per-token queries, " +
                      std::to_string(s.n_prefill_tiles) + " prefill tiles)"};
      const bool enough = counters != nullptr && (uint64_t)counters->numel() >= count;
      if (!enough && (counters == nullptr || counters_grow)) {
        meanwhile.reset();
        return PyLong_FromUnsignedLongLong(count);
      }
      if (!enough || counters->scalar_type() != at::kInt || counters->device() != dev)
        throw Refused{"counters must be an int32 device tensor of at least " + std::to_string(count) + " entries"};
      if (ws == nullptr) {
        room = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
        ws = &room;
      }
      s.workspace = ws->data_ptr();
      s.workspace_bytes = need;
      s.counters = words(counters);
    }
    const hipStream_t stream = reinterpret_cast<hipStream_t>(handle);
    checked(window == 0 ? call(&s, stream) : window_call(&s, (int32_t)window, (int32_t)sinks, stream));
    meanwhile.reset();
    return answer();
  });
}

// pages(kind, the library's function, ns_kv_last_error, ns_kv_pool address, device index, list, other list or None, window,
//       sinks, stream handle) -> None, or False where a list is not a contiguous int32 tensor of one dimension on the
// device, for the caller to make it one.  kind 0: ns_kv_free; 1: ns_kv_extend or ns_kv_fork; 2: ns_kv_release.
PyObject* pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments(n, 10)) return nullptr;
  return guarded(g_store_error, [&]() -> PyObject* {
    const int64_t kind = number(a[0]), index = number(a[4]);
    const ns_kv_pool* pool = function<const ns_kv_pool*>(a[3]);
    const at::Tensor* list[2] = {nullptr, nullptr};
    for (int i = 0; i < (kind == 1 ? 2 : 1); ++i) {
      if (!THPVariable_Check(a[5 + i])) Py_RETURN_FALSE;
      list[i] = &THPVariable_Unpack(a[5 + i]);
      if (list[i]->scalar_type() != at::kInt || list[i]->dim() != 1 || !list[i]->is_cuda() ||
          list[i]->get_device() != index || !list[i]->is_contiguous())
        Py_RETURN_FALSE;
    }
    if (kind == 1 && list[0]->numel() != list[1]->numel())
      throw Refused{"the two lists must be as many (got " + std::to_string(list[0]->numel()) + " and " +
                    std::to_string(list[1]->numel()) + ")"};
    if (list[0]->numel() > INT32_MAX) throw Refused{"the list is too long"};
    const int32_t count = (int32_t)list[0]->numel();
    const int64_t window = number(a[7]), sinks = number(a[8]);
    const hipStream_t stream = reinterpret_cast<hipStream_t>(number(a[9]));
    void* const call = PyLong_AsVoidPtr(a[1]);
    const auto why = function<decltype(&ns_kv_last_error)>(a[2]);
    std::optional<Unlocked> meanwhile(std::in_place);
    const int rc = kind == 0   ? reinterpret_cast<decltype(&ns_kv_free)>(call)(pool, words(list[0]), count, stream)
                   : kind == 1 ? reinterpret_cast<decltype(&ns_kv_extend)>(call)(pool, words(list[0]), words(list[1]), count, stream)
                               : reinterpret_cast<decltype(&ns_kv_release)>(call)(pool, words(list[0]), count, (int32_t)window,
                                                                                  (int32_t)sinks, stream);
    if (rc != 0) throw Refused{why()};
    meanwhile.reset();
    Py_RETURN_NONE;
  });
}

// ---- mx.py ----------------------------------------------------------------------------------------------------

int mx_type(const at::Tensor& t, const char* name) {
  const at::ScalarType type = t.scalar_type();
  if (type == at::kBFloat16) return NS_MX_BF16;
  if (type == at::kHalf) return NS_MX_F16;
  if (type == at::kFloat) return NS_MX_F32;
  throw Refused{std::string(name) + ": unsupported dtype " + c10::toString(type) + " (float32, bfloat16, float16)"};
}
at::ScalarType torch_type(int64_t type) { return type == NS_MX_F32 ? at::kFloat : type == NS_MX_BF16 ? at::kBFloat16 : at::kHalf; }

// The bytes of a row (what follows the first dimension), and the bytes from row to row.
int64_t row_bytes(const at::Tensor& t) {
  int64_t last = 0;
  for (int64_t i = 1; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  return (last + 1) * (int64_t)t.element_size();
}
int64_t pitch(const at::Tensor& t) { return t.stride(0) * (int64_t)t.element_size(); }

// Whether two tensors of at least one row have no byte in common: their ranges do not meet, or their rows lie beside
// each other in wider ones.  (What lies apart in other ways is not seen.)
bool apart(const at::Tensor& a, const at::Tensor& b) {
  const auto at = [](const at::Tensor& t) { return reinterpret_cast<intptr_t>(t.data_ptr()); };
  const int64_t pa = pitch(a), pb = pitch(b), ra = row_bytes(a), rb = row_bytes(b);
  const intptr_t a0 = at(a), b0 = at(b), a1 = a0 + (a.size(0) - 1) * pa + ra, b1 = b0 + (b.size(0) - 1) * pb + rb;
  if (a1 <= b0 || b1 <= a0) return true;
  if (pa != pb || pa <= 0) return false;
  const int64_t d = (int64_t)(((b0 - a0) % pa + pa) % pa);   // b's rows begin so far behind a's
  return d >= ra && d + rb <= pa;
}
bool same_view(const at::Tensor& a, const at::Tensor& b) {
  return a.data_ptr() == b.data_ptr() && a.sizes() == b.sizes() && a.strides() == b.strides() && a.scalar_type() == b.scalar_type();
}

// A new tensor on the current device (which is `like`'s: the caller has made it so), of torch's allocator for it, as at::empty
// makes it on its way through the dispatcher.
at::Tensor fresh(const at::Tensor& like, at::IntArrayRef size, at::ScalarType type) {
  static c10::Allocator* const allocator = at::empty({16}, like.options()).storage().allocator();
  if (allocator == nullptr) return at::empty(size, like.options().dtype(type));
  return at::detail::empty_generic(size, allocator, c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt);
}

struct Written {   // a tensor that a call writes, and one that it reads or writes
  const char* name;
  const at::Tensor* t;
};
// Rows that do not overlap within the tensor, no byte of what else is written, and what is read only as a whole and with `in_place`.
void check_written(std::initializer_list<Written> out, std::initializer_list<Written> in, bool in_place) {
  for (const Written& w : out) {
    if (w.t == nullptr) continue;
    const at::Tensor& t = *w.t;
    if ((t.dim() == 3 && t.size(1) > 1 && t.stride(1) < t.size(2)) || (t.size(0) > 1 && pitch(t) < row_bytes(t)))
      throw Refused{std::string(w.name) + "'s rows overlap"};
    for (const Written& o : out)
      if (o.t != nullptr && &o != &w && !apart(t, *o.t))
        throw Refused{std::string(w.name) + " and " + o.name + " overlap"};
    for (const Written& r : in)
      if (r.t != nullptr && !apart(t, *r.t) && !(in_place && same_view(t, *r.t)))
        throw Refused{std::string(w.name) + " overlaps " + r.name};
  }
}

// MX rows: codes (rows, k) float8_e4m3fn or (rows, k / 2) float4_e2m1fn_x2, scales (rows, k / 32) float8_e8m0fnu.  Returns k.
int64_t mx_rows_of(const at::Tensor& codes, const at::Tensor& scales, const std::string& name, ns_mx_rows* to) {
  const at::ScalarType type = codes.scalar_type();
  if (type != at::kFloat8_e4m3fn && type != at::kFloat4_e2m1fn_x2)
    throw Refused{name + ": codes must be float8_e4m3fn or float4_e2m1fn_x2, not " + c10::toString(type)};
  if (scales.scalar_type() != at::kFloat8_e8m0fnu)
    throw Refused{name + ": scales must be float8_e8m0fnu, not " + c10::toString(scales.scalar_type())};
  if (codes.dim() != 2 || scales.dim() != 2 || codes.size(0) != scales.size(0))
    throw Refused{name + ": codes " + shape_of(codes) + " and scales " + shape_of(scales) + " must be as many rows"};
  const int64_t k = codes.size(1) * (type == at::kFloat4_e2m1fn_x2 ? 2 : 1);
  if (k == 0 || k % NS_MX_ROW_ALIGN != 0 || scales.size(1) != k / 32)
    throw Refused{name + ": rows must be padded to a multiple of 128 values with a scale for every 32 (mx_tensor lays them out); got codes " +
                  shape_of(codes) + " and scales " + shape_of(scales)};
  if (codes.device() != scales.device()) throw Refused{name + ": codes and scales must be on one device"};
  if (codes.stride(1) != 1 || scales.stride(1) != 1) throw Refused{name + ": codes and scales must have a unit stride along the row"};
  if (codes.size(0) > 1 && (codes.stride(0) % 16 != 0 || scales.stride(0) % 4 != 0 || codes.stride(0) < codes.size(1) ||
                            scales.stride(0) < scales.size(1)))
    throw Refused{name + ": code rows must lie behind each other at multiples of 16 bytes, scale rows at multiples of 4"};
  to->codes = codes.data_ptr();
  to->scales = static_cast<uint8_t*>(scales.data_ptr());
  to->stride_codes = codes.size(0) > 1 ? codes.stride(0) : codes.size(1);
  to->stride_scales = codes.size(0) > 1 ? scales.stride(0) : scales.size(1);
  to->format = type == at::kFloat4_e2m1fn_x2 ? NS_MX_FP4 : NS_MX_FP8;
  return k;
}

const char* const kNoStride = " must have a unit stride along the row";

// What a call returns: a tensor, or the codes and scales of MX rows; given by the caller or made here.
struct Result {
  PyObject *given, *given_scales;
  int64_t format;
  at::Tensor made, made_scales;
  const at::Tensor *out = nullptr, *scales = nullptr;

  // of n rows shaped like `like`'s, checked where given
  Result(PyObject* out0, PyObject* scales0, int64_t format, const at::Tensor& like, int64_t n)
      : given(out0), given_scales(scales0), format(format) {
    if (format != 0 && format != NS_MX_FP4 && format != NS_MX_FP8) throw Refused{"format must be None, \"mxfp4\" or \"mxfp8\""};
    out = tensor(out0, "out");
    scales = tensor(scales0, "out's scales");
    if (!out != !scales && format != 0) throw Refused{"out must hold codes and scales"};
    if (format == 0 && scales != nullptr) throw Refused{"out must be a tensor where no format is given"};
    if (out == nullptr) return;
    if (out->device() != like.device()) throw Refused{"out must be on the input's device"};
    if (format == 0) {
      bool fits = out->dim() == like.dim() && out->size(0) == n && out->scalar_type() == like.scalar_type();
      for (int64_t i = 1; fits && i < like.dim(); ++i) fits = out->size(i) == like.size(i);
      if (!fits) throw Refused{"out " + shape_of(*out) + " must have the result's shape and dtype"};
      if (out->stride(-1) != 1 && out->size(-1) > 1) throw Refused{std::string("out") + kNoStride};
    } else {
      ns_mx_rows r;
      const int64_t k = mx_rows_of(*out, *scales, "out", &r);
      if (r.format != format || out->size(0) != n || k != padded(like))
        throw Refused{"out " + shape_of(*out) + " must have the result's format and shape"};
    }
  }
  static int64_t padded(const at::Tensor& like) {
    return (like.size(-1) + NS_MX_ROW_ALIGN - 1) / NS_MX_ROW_ALIGN * NS_MX_ROW_ALIGN;
  }
  void make(const at::Tensor& like, int64_t n) {   // without Python's lock
    if (out != nullptr) return;
    if (format == 0) {
      const int64_t size[] = {n, like.size(1), like.dim() == 3 ? like.size(2) : 1};
      made = fresh(like, at::IntArrayRef(size, like.dim()), like.scalar_type());
    } else {
      const int64_t k = padded(like), codes[] = {n, format == NS_MX_FP4 ? k / 2 : k}, blocks[] = {n, k / 32};
      made = fresh(like, codes, format == NS_MX_FP4 ? at::kFloat4_e2m1fn_x2 : at::kFloat8_e4m3fn);
      made_scales = fresh(like, blocks, at::kFloat8_e8m0fnu);
      scales = &made_scales;
    }
    out = &made;
  }
  void pack(void** plain, ns_mx_rows* mx) const {
    if (format == 0) *plain = out->data_ptr();
    else mx_rows_of(*out, *scales, "out", mx);
  }
  PyObject* answer() const {
    const auto one = [](const at::Tensor& made, PyObject* given) {
      if (made.defined()) return THPVariable_Wrap(made);
      Py_INCREF(given);
      return given;
    };
    PyObject* o = one(made, given);
    if (format == 0 || o == nullptr) return o;
    PyObject* s = one(made_scales, given_scales);
    PyObject* both = s == nullptr ? nullptr : PyTuple_Pack(2, o, s);
    Py_DECREF(o);
    Py_XDECREF(s);
    return both;
  }
};

const int64_t* picked(const at::Tensor* rows, const at::Tensor& x) {
  if (rows == nullptr) return nullptr;
  if (rows->scalar_type() != at::kLong || rows->dim() != 1 || !rows->is_contiguous() || rows->device() != x.device())
    throw Refused{"rows must be a contiguous int64 tensor of one dimension on the input's device"};
  return static_cast<const int64_t*>(rows->data_ptr());
}
void check_cols(const at::Tensor& x, const char* name, int64_t most) {
  if (x.size(-1) < 1 || x.size(-1) > most)
    throw Refused{std::string(name) + " must have 1 to " + std::to_string(most) + " columns, not " + std::to_string(x.size(-1))};
  if (x.numel() > 0 && x.stride(-1) != 1 && x.size(-1) > 1) throw Refused{std::string(name) + kNoStride};
}
void check_like(const at::Tensor* t, const char* name, const at::Tensor& x, const char* of, int64_t n) {
  if (t == nullptr) return;
  bool fits = t->dim() == x.dim() && t->size(0) == n;
  for (int64_t i = 1; fits && i < x.dim(); ++i) fits = t->size(i) == x.size(i);
  if (!fits || t->scalar_type() != x.scalar_type() || t->device() != x.device())
    throw Refused{std::string(name) + " " + shape_of(*t) + " must have the shape, dtype and device of " + of + " " + shape_of(x)};
  if (t->numel() > 0 && t->stride(-1) != 1 && t->size(-1) > 1) throw Refused{std::string(name) + kNoStride};
}

// rms_norm(ns_mx_rms_norm, ns_mx_last_error, x, weight, eps, residual, sum_out, rows, format, out, out's scales, stream
//          handle) -> out, or codes and scales
PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments(n, 12)) return nullptr;
  return guarded(g_mx_error, [&]() -> PyObject* {
    const at::Tensor &x = needed(a[2], "x"), &weight = needed(a[3], "weight");
    const double eps = PyFloat_AsDouble(a[4]);
    if (eps == -1.0 && PyErr_Occurred()) throw Refused{""};
    const at::Tensor *residual = tensor(a[5], "residual"), *sum = tensor(a[6], "sum_out"), *rows = tensor(a[7], "rows");
    const int64_t format = number(a[8]), handle = number(a[11]);
    ns_mx_norm_args s = {};
    s.dtype = mx_type(x, "x");
    if (x.dim() != 2 && x.dim() != 3) throw Refused{"x must have two or three dimensions, not " + std::to_string(x.dim())};
    check_cols(x, "x", 1 << 30);
    if (x.dim() == 3 && x.size(1) > INT32_MAX) throw Refused{"x has too many heads"};
    if (x.dim() == 3 && rows != nullptr) throw Refused{"rows needs an x of two dimensions"};
    if (x.dim() == 3 && format != 0) throw Refused{"a format needs an x of two dimensions"};
    if (weight.dim() != 1 || weight.size(0) != x.size(-1) || weight.device() != x.device() ||
        (weight.scalar_type() != x.scalar_type() && weight.scalar_type() != at::kFloat))
      throw Refused{"weight " + shape_of(weight) + " must have x's columns, dtype (or float32) and device"};
    if (weight.size(0) > 1 && weight.stride(0) != 1) throw Refused{"weight must be contiguous"};
    if (!(eps >= 0.0)) throw Refused{"eps must be at least 0"};
    s.rows = picked(rows, x);
    s.n_x = x.size(0);
    s.n = rows != nullptr ? rows->size(0) : s.n_x;
    if (s.n > 0 && s.n_x == 0) throw Refused{"rows of an empty x"};
    check_like(residual, "residual", x, "x", s.n_x);
    check_like(sum, "sum_out", x, "the result: x", s.n);
    Result r(a[9], a[10], format, x, s.n);
    if (!x.is_cuda()) throw Refused{"rms_norm_hip needs device tensors"};
    const bool any = s.n > 0 && x.numel() > 0;
    if (any) check_written({{"out", r.out}, {"out's scales", r.scales}, {"sum_out", sum}},
                           {{"x", &x}, {"residual", residual}, {"weight", &weight}, {"rows", rows}}, rows == nullptr);
    const auto call = function<decltype(&ns_mx_rms_norm)>(a[0]);
    const auto why = function<decltype(&ns_mx_last_error)>(a[1]);
    std::optional<Unlocked> meanwhile(std::in_place);
    r.make(x, s.n);
    if (any) {
      r.pack(&s.out, &s.out_mx);
      s.x = x.data_ptr();
      s.residual = at_of(residual);
      s.weight = weight.data_ptr();
      s.weight_dtype = weight.scalar_type() == at::kFloat ? NS_MX_F32 : s.dtype;
      s.sum = at_of(sum);
      s.heads = x.dim() == 3 ? (int32_t)x.size(1) : 1;
      s.cols = (int32_t)x.size(-1);
      s.eps = (float)eps;
      const auto strides = [&](const at::Tensor* t, int64_t* row, int64_t* head) {
        if (t == nullptr) return;
        *row = t->stride(0);
        *head = t->dim() == 3 ? t->stride(1) : 0;
      };
      strides(&x, &s.stride_x, &s.stride_x_head);
      strides(residual, &s.stride_residual, &s.stride_residual_head);
      strides(sum, &s.stride_sum, &s.stride_sum_head);
      if (format == 0) strides(r.out, &s.stride_out, &s.stride_out_head);
      if (call(&s, reinterpret_cast<hipStream_t>(handle)) != 0) throw Refused{why()};
    }
    meanwhile.reset();
    return r.answer();
  });
}

// silu_mul(ns_mx_silu_mul, ns_mx_last_error, gate, up, None, format, out, out's scales, stream handle) and
// quantize(ns_mx_quantize, ns_mx_last_error, x, None, rows, format, out, out's scales, stream handle) -> out, or codes and
// scales.  ns_mx_silu_mul and ns_mx_quantize are of one type.
PyObject* gate(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments(n, 9)) return nullptr;
  return guarded(g_mx_error, [&]() -> PyObject* {
    const bool gated = a[3] != Py_None;
    const char* name = gated ? "gate" : "x";
    const at::Tensor& x = needed(a[2], name);
    const at::Tensor *up = tensor(a[3], "up"), *rows = tensor(a[4], "rows");
    const int64_t format = number(a[5]), handle = number(a[8]);
    ns_mx_gate_args s = {};
    s.dtype = mx_type(x, name);
    if (x.dim() != 2) throw Refused{std::string(name) + " must have two dimensions, not " + std::to_string(x.dim())};
    check_cols(x, name, 1 << 26);
    check_like(up, "up", x, "gate", x.size(0));
    if (!gated && format == 0) throw Refused{"format must be \"mxfp4\" or \"mxfp8\""};
    s.rows = picked(rows, x);
    s.n_x = x.size(0);
    s.n = rows != nullptr ? rows->size(0) : s.n_x;
    if (s.n > 0 && s.n_x == 0) throw Refused{"rows of an empty x"};
    Result r(a[6], a[7], format, x, s.n);
    if (!x.is_cuda()) throw Refused{gated ? "silu_mul_hip needs device tensors" : "quantize_mx_hip needs device tensors"};
    if (s.n > 0) check_written({{"out", r.out}, {"out's scales", r.scales}}, {{name, &x}, {"up", up}, {"rows", rows}}, true);
    const auto call = function<decltype(&ns_mx_silu_mul)>(a[0]);
    const auto why = function<decltype(&ns_mx_last_error)>(a[1]);
    std::optional<Unlocked> meanwhile(std::in_place);
    r.make(x, s.n);
    if (s.n > 0) {
      r.pack(&s.out, &s.out_mx);
      s.gate = x.data_ptr();
      s.up = at_of(up);
      s.stride_gate = x.stride(0);
      s.stride_up = up != nullptr ? up->stride(0) : 0;
      s.stride_out = format == 0 ? r.out->stride(0) : 0;
      s.cols = (int32_t)x.size(1);
      if (call(&s, reinterpret_cast<hipStream_t>(handle)) != 0) throw Refused{why()};
    }
    meanwhile.reset();
    return r.answer();
  });
}

// dequantize(ns_mx_dequantize, ns_mx_last_error, codes, scales, cols or -1, dtype (NS_MX_*), out, stream handle) -> out
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments(n, 8)) return nullptr;
  return guarded(g_mx_error, [&]() -> PyObject* {
    const at::Tensor &codes = needed(a[2], "codes"), &scales = needed(a[3], "scales");
    int64_t cols = number(a[4]);
    const int64_t dtype = number(a[5]), handle = number(a[7]);
    const at::Tensor* out = tensor(a[6], "out");
    ns_mx_rows r;
    const int64_t k = mx_rows_of(codes, scales, "t", &r), rows = codes.size(0);
    if (cols == -1) cols = k;
    if (cols < 1 || cols > k || cols > 1 << 26)
      throw Refused{"cols must lie in 1 .. " + std::to_string(k) + ", the rows' width, not " + std::to_string(cols)};
    if (out != nullptr) {
      if (out->dim() != 2 || out->size(0) != rows || out->size(1) != cols || out->scalar_type() != torch_type(dtype) ||
          out->device() != codes.device())
        throw Refused{"out " + shape_of(*out) + " must have the result's shape, dtype and device"};
      if (out->stride(1) != 1 && cols > 1) throw Refused{std::string("out") + kNoStride};
    }
    if (!codes.is_cuda()) throw Refused{"dequantize_mx_hip needs device tensors"};
    if (rows > 0) check_written({{"out", out}}, {{"codes", &codes}, {"scales", &scales}}, false);
    const auto call = function<decltype(&ns_mx_dequantize)>(a[0]);
    const auto why = function<decltype(&ns_mx_last_error)>(a[1]);
    std::optional<Unlocked> meanwhile(std::in_place);
    at::Tensor made;
    if (out == nullptr) {
      const int64_t size[] = {rows, cols};
      made = fresh(codes, size, torch_type(dtype));
      out = &made;
    }
    if (rows > 0 && call(&r, rows, (int32_t)cols, out->data_ptr(), out->stride(0), (int32_t)dtype,
                         reinterpret_cast<hipStream_t>(handle)) != 0)
      throw Refused{why()};
    meanwhile.reset();
    if (made.defined()) return THPVariable_Wrap(made);
    Py_INCREF(a[6]);
    return a[6];
  });
}

// linear(ns_mx_linear, ns_mx_last_error, x's codes, scales, the weight's codes, scales, dtype (NS_MX_*), out, stream handle)
// -> out
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments(n, 9)) return nullptr;
  return guarded(g_mx_error, [&]() -> PyObject* {
    const at::Tensor &xc = needed(a[2], "x's codes"), &xs = needed(a[3], "x's scales"), &wc = needed(a[4], "weight's codes"),
                     &ws = needed(a[5], "weight's scales");
    const int64_t dtype = number(a[6]), handle = number(a[8]);
    const at::Tensor* out = tensor(a[7], "out");
    ns_mx_linear_args s = {};
    const int64_t k = mx_rows_of(xc, xs, "x", &s.x), kw = mx_rows_of(wc, ws, "weight", &s.weight);
    if (s.weight.format != NS_MX_FP4) throw Refused{"weight: codes must be float4_e2m1fn_x2"};
    if (k != kw) throw Refused{"x's rows of " + std::to_string(k) + " values do not match the weight's of " + std::to_string(kw)};
    if (k > INT32_MAX) throw Refused{"rows are too wide"};
    if (xc.device() != wc.device()) throw Refused{"x and weight must be on one device"};
    s.m = xc.size(0);
    s.n = wc.size(0);
    if (out != nullptr) {
      if (out->dim() != 2 || out->size(0) != s.m || out->size(1) != s.n || out->scalar_type() != torch_type(dtype) ||
          out->device() != xc.device())
        throw Refused{"out " + shape_of(*out) + " must have the result's shape, dtype and device"};
      if (out->stride(1) != 1 && s.n > 1) throw Refused{std::string("out") + kNoStride};
    }
    if (!xc.is_cuda()) throw Refused{"mx_linear_hip needs device tensors"};
    const bool any = s.m > 0 && s.n > 0;
    if (any) check_written({{"out", out}}, {{"x's codes", &xc}, {"x's scales", &xs}, {"weight's codes", &wc}, {"weight's scales", &ws}}, false);
    const auto call = function<decltype(&ns_mx_linear)>(a[0]);
    const auto why = function<decltype(&ns_mx_last_error)>(a[1]);
    std::optional<Unlocked> meanwhile(std::in_place);
    at::Tensor made;
    if (out == nullptr) {
      const int64_t size[] = {s.m, s.n};
      made = fresh(xc, size, torch_type(dtype));
      out = &made;
    }
    if (any) {
      s.out = out->data_ptr();
      s.stride_out = out->stride(0);
      s.k = (int32_t)k;
      s.dtype = (int32_t)dtype;
      if (call(&s, reinterpret_cast<hipStream_t>(handle)) != 0) throw Refused{why()};
    }
    meanwhile.reset();
    if (made.defined()) return THPVariable_Wrap(made);
    Py_INCREF(a[7]);
    return a[7];
  });
}

// set_errors(attention's, the cache's[, mx's]): None leaves one as it is
PyObject* set_errors(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3 && !arguments(n, 2)) return nullptr;
  PyObject** to[] = {&g_attention_error, &g_store_error, &g_mx_error};
  for (int i = 0; i < n; ++i)
    if (a[i] != Py_None) {
      Py_INCREF(a[i]);
      Py_XDECREF(*to[i]);
      *to[i] = a[i];
    }
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"store", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(store)), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL, nullptr},
    {"pages", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(pages)), METH_FASTCALL, nullptr},
    {"rms_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rms_norm)), METH_FASTCALL, nullptr},
    {"gate", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gate)), METH_FASTCALL, nullptr},
    {"dequantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dequantize)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear)), METH_FASTCALL, nullptr},
    {"set_errors", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(set_errors)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_ns_host", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__ns_host() { return PyModule_Create(&g_module); }
