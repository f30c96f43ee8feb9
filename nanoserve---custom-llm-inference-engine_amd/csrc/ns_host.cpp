// The host side of the attention's, the cache store's and the page pool's calls: argument checks, the packing of the C ABI's structs and
// the call, which in Python took 8 to 12 us of a call whose kernel takes 4.  The modules paged_attention.py and
// kv_cache.py hold the interfaces and say what the arguments mean; the kernels stay behind their C ABI, whose functions
// come in as addresses.

#include <Python.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>

#include <exception>
#include <optional>
#include <string>
#include <utility>

#include "ns_kv_cache.h"
#include "ns_paged_attention.h"

namespace {

struct Refused {
  std::string why;
};

PyObject* g_attention_error = nullptr;   // exception classes, set once by the modules
PyObject* g_store_error = nullptr;

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

PyObject* set_errors(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!arguments(n, 2)) return nullptr;
  PyObject** to[] = {&g_attention_error, &g_store_error};
  for (int i = 0; i < 2; ++i)
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
    {"set_errors", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(set_errors)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_ns_host", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__ns_host() { return PyModule_Create(&g_module); }
