// The plain calls of gemv, qk_norm_rope, the cache's operators and paged_attention without the Python
// wrappers' cost: arguments are looked at and results allocated here.  A call that is not as it should be, or
// has an option that is not known here, gets None and goes through the wrapper, which says what is wrong.  (A
// tensor's checks cost some 1 us in Python and an allocation 2 us; one launch is 2.3 us.)  Built where torch's
// headers and a C++ compiler are; the wrappers work without it.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>

#include "../../include/chord_b200.h"

namespace {

constexpr int kMaxDevices = 64;
constexpr int kMaxStreams = 16;
constexpr int64_t kMaxRoutedRows = 65535;  // of gemv, rows with an expert each

struct Entries {
  decltype(&chord_b200_gemv) gemv;
  decltype(&chord_b200_qk_norm_rope) qk_norm_rope;
  decltype(&chord_b200_qk_norm_rope_write) qk_norm_rope_write;
  decltype(&chord_b200_cache_write) cache_write;
  decltype(&chord_b200_cache_read) cache_read;
  decltype(&chord_b200_paged_attention) paged_attention;
  decltype(&chord_b200_paged_attention_workspace_bytes) workspace_bytes;
} entries;

// What the wrappers keep for a device: its status word and the lock buffers of its streams.  (Under the
// interpreter's lock.)
struct Device {
  int32_t* status = nullptr;
  struct {
    void* stream = nullptr;
    int32_t* words = nullptr;
    int64_t count = 0;
  } locks[kMaxStreams];
} devices[kMaxDevices];

PyObject* none() { Py_RETURN_NONE; }

const at::Tensor* tensor(PyObject* o, at::ScalarType type, int64_t dims) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.scalar_type() == type && t.dim() == dims && t.is_cuda() && t.layout() == at::kStrided ? &t : nullptr;
}

// The device of a first tensor, if calls may go to it from here.
int device_of(const at::Tensor& t) {
  const int index = t.get_device();
  return index >= 0 && index < kMaxDevices && devices[index].status != nullptr && index == c10::cuda::current_device() ? index : -1;
}

bool aligned(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0; }

// [tokens, heads, dim] with rows on 16-byte boundaries; heads < 0: any but none.
bool rows(const at::Tensor* t, int device, int64_t tokens, int64_t heads, int64_t dim) {
  return t != nullptr && t->get_device() == device && t->size(0) == tokens && (heads < 0 ? t->size(1) > 0 : t->size(1) == heads) &&
         t->size(2) == dim && t->stride(2) == 1 && t->stride(0) % 8 == 0 && t->stride(1) % 8 == 0 && t->stride(0) >= 0 &&
         t->stride(1) >= 0 && aligned(*t);
}

const int32_t* ints(PyObject* o, int device, int64_t count) {
  const at::Tensor* t = tensor(o, at::kInt, 1);
  return t != nullptr && t->get_device() == device && t->size(0) == count && (count <= 1 || t->stride(0) == 1) ? t->const_data_ptr<int32_t>() : nullptr;
}

at::Tensor empty(at::IntArrayRef sizes, const at::Tensor& like, at::ScalarType type = at::kBFloat16) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }

bool integer(PyObject* o, int64_t* value) {
  if (!PyLong_CheckExact(o)) return false;
  *value = PyLong_AsLongLong(o);
  if (*value == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

bool number(PyObject* o, double* value) {
  if (!PyFloat_CheckExact(o)) return false;
  *value = PyFloat_AS_DOUBLE(o);
  return std::isfinite(*value);
}

// A KVCache's (descriptor's address, device): as the wrappers made and checked them.
bool cache_of(PyObject* address, PyObject* device, const chord_b200_kv_cache** cache, int* index) {
  int64_t at, on;
  if (!integer(address, &at) || !integer(device, &on) || at == 0 || on < 0 || on >= kMaxDevices) return false;
  if (devices[on].status == nullptr || on != c10::cuda::current_device()) return false;
  *cache = reinterpret_cast<const chord_b200_kv_cache*>(at);
  *index = static_cast<int>(on);
  return true;
}

PyObject* pair(at::Tensor&& a, at::Tensor&& b) {
  PyObject* x = THPVariable_Wrap(std::move(a));
  PyObject* y = THPVariable_Wrap(std::move(b));
  PyObject* both = x != nullptr && y != nullptr ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return both;
}

// Without the interpreter's lock: an allocation may wait for the device and a launch for room in its queue, behind
// a host function that itself wants the lock.
class Unlocked {
 public:
  Unlocked() : state_(PyEval_SaveThread()) {}
  ~Unlocked() { PyEval_RestoreThread(state_); }
  Unlocked(const Unlocked&) = delete;
  Unlocked& operator=(const Unlocked&) = delete;

 private:
  PyThreadState* state_;
};

using Call = PyObject* (*)(PyObject*, PyObject* const*, Py_ssize_t);

// A C++ exception (out of memory) ends here; the wrapper then meets it itself.
template <Call call>
PyObject* guarded(PyObject* self, PyObject* const* a, Py_ssize_t count) {
  try {
    return call(self, a, count);
  } catch (...) {
    PyErr_Clear();
    return none();
  }
}

// gemv(x, packed, scale, n, k, experts, expert_ids, top_k, expert_base)
PyObject* gemv(PyObject*, PyObject* const* a, Py_ssize_t count) {
  int64_t n, k, experts, top_k, base;
  if (count != 9 || !integer(a[3], &n) || !integer(a[4], &k) || !integer(a[5], &experts) || !integer(a[7], &top_k) ||
      !integer(a[8], &base))
    return none();
  const at::Tensor *x = tensor(a[0], at::kBFloat16, 2), *packed = tensor(a[1], at::kInt, 3), *scale = tensor(a[2], at::kBFloat16, 3);
  if (x == nullptr || packed == nullptr || scale == nullptr) return none();
  const int device = device_of(*x);
  if (device < 0 || packed->get_device() != device || scale->get_device() != device || !packed->is_contiguous() ||
      !scale->is_contiguous() || packed->size(0) != experts || packed->size(1) != k / 16 || packed->size(2) != 2 * n ||
      scale->size(0) != experts || scale->size(1) != k / 32 || scale->size(2) != n || x->size(1) != k)
    return none();
  int64_t rows = x->size(0);
  const int64_t stride = rows > 1 ? x->stride(0) : k;
  if (rows == 0 || x->stride(1) != 1 || stride < k || stride % 2 != 0 || (reinterpret_cast<uintptr_t>(x->const_data_ptr()) & 3) != 0 ||
      top_k < 1 || top_k > kMaxRoutedRows || base < 0)
    return none();
  const int32_t* ids = nullptr;
  if (a[6] == Py_None) {
    if (experts != 1 || top_k != 1 || base != 0 || rows > 16) return none();
  } else {
    if (!THPVariable_Check(a[6])) return none();
    const at::Tensor& t = THPVariable_Unpack(a[6]);
    rows *= top_k;
    if (t.scalar_type() != at::kInt || !t.is_cuda() || t.get_device() != device || !t.is_contiguous() || t.numel() != rows || rows > kMaxRoutedRows)
      return none();
    ids = t.const_data_ptr<int32_t>();
  }
  at::Tensor out;
  int rc;
  {
    const Unlocked unlocked;
    out = empty({rows, n}, *x);
    rc = entries.gemv(x->const_data_ptr(), stride, static_cast<const int32_t*>(packed->const_data_ptr()), scale->const_data_ptr(), ids,
                      out.mutable_data_ptr(), rows, n, k, experts, top_k, base, stream_of(device));
  }
  return rc ? none() : THPVariable_Wrap(std::move(out));
}

struct Rotation {
  const at::Tensor *q, *k, *q_weight, *k_weight, *table;
  const int32_t* positions;
  int device;
  int64_t tokens, dim;
  double eps;
  bool interleaved;
};

// q, k, q_weight, k_weight, cos_sin, positions, eps, interleaved; kv_heads < 0: any.
bool rotation(PyObject* const* a, int64_t kv_heads, Rotation* r) {
  r->q = tensor(a[0], at::kBFloat16, 3);
  r->k = tensor(a[1], at::kBFloat16, 3);
  r->q_weight = tensor(a[2], at::kBFloat16, 1);
  r->k_weight = tensor(a[3], at::kBFloat16, 1);
  r->table = tensor(a[4], at::kFloat, 2);
  if (r->q == nullptr || r->k == nullptr || r->q_weight == nullptr || r->k_weight == nullptr || r->table == nullptr) return false;
  r->device = device_of(*r->q);
  r->tokens = r->q->size(0);
  r->dim = r->q->size(2);
  if (r->device < 0 || r->tokens == 0 || !rows(r->q, r->device, r->tokens, -1, r->dim) || !rows(r->k, r->device, r->tokens, kv_heads, r->dim)) return false;
  for (const at::Tensor* w : {r->q_weight, r->k_weight}) {
    if (w->get_device() != r->device || w->size(0) != r->dim || w->stride(0) != 1 || !aligned(*w)) return false;
  }
  const int64_t rotary = r->table->size(1);
  if (r->dim % 16 != 0 || r->dim > 256 || r->table->get_device() != r->device || r->table->size(0) == 0 || rotary % 16 != 0 ||
      rotary > r->dim || rotary == 0 || !r->table->is_contiguous() || !aligned(*r->table))
    return false;
  r->positions = ints(a[5], r->device, r->tokens);
  if (r->positions == nullptr || !number(a[6], &r->eps) || r->eps < 0 || !PyBool_Check(a[7])) return false;
  r->interleaved = a[7] == Py_True;
  return true;
}

// qk_norm_rope(q, k, q_weight, k_weight, cos_sin, positions, eps, interleaved)
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t count) {
  Rotation r;
  if (count != 8 || !rotation(a, -1, &r)) return none();
  int32_t* const status = devices[r.device].status;
  at::Tensor q_out, k_out;
  int rc;
  {
    const Unlocked unlocked;
    q_out = empty(r.q->sizes(), *r.q), k_out = empty(r.k->sizes(), *r.k);
    rc = entries.qk_norm_rope(r.q->const_data_ptr(), r.q->stride(0), r.q->stride(1), r.k->const_data_ptr(), r.k->stride(0), r.k->stride(1),
                              r.q_weight->const_data_ptr(), r.k_weight->const_data_ptr(), r.table->const_data_ptr<float>(),
                              r.table->size(0), r.table->size(1), r.interleaved, r.positions, q_out.mutable_data_ptr(),
                              k_out.mutable_data_ptr(), r.tokens, r.q->size(1), r.k->size(1), r.dim, status, r.eps,
                              stream_of(r.device));
  }
  return rc ? none() : pair(std::move(q_out), std::move(k_out));
}

// qk_norm_rope_write(q, k, q_weight, k_weight, cos_sin, positions, eps, interleaved, v, cache, device, slots)
PyObject* qk_norm_rope_write(PyObject*, PyObject* const* a, Py_ssize_t count) {
  const chord_b200_kv_cache* cache;
  int device;
  Rotation r;
  if (count != 12 || !cache_of(a[9], a[10], &cache, &device) || !rotation(a, cache->heads, &r) || r.device != device ||
      r.dim != cache->head_dim)
    return none();
  const at::Tensor* v = tensor(a[8], at::kBFloat16, 3);
  const int32_t* slots = ints(a[11], device, r.tokens);
  if (!rows(v, device, r.tokens, cache->heads, r.dim) || slots == nullptr) return none();
  int32_t* const status = devices[device].status;
  at::Tensor q_out;
  int rc;
  {
    const Unlocked unlocked;
    q_out = empty(r.q->sizes(), *r.q);
    rc = entries.qk_norm_rope_write(r.q->const_data_ptr(), r.q->stride(0), r.q->stride(1), r.k->const_data_ptr(), r.k->stride(0),
                                    r.k->stride(1), v->const_data_ptr(), v->stride(0), v->stride(1), r.q_weight->const_data_ptr(),
                                    r.k_weight->const_data_ptr(), r.table->const_data_ptr<float>(), r.table->size(0), r.table->size(1),
                                    r.interleaved, r.positions, q_out.mutable_data_ptr(), cache, slots, r.tokens, r.q->size(1),
                                    status, r.eps, stream_of(device));
  }
  return rc ? none() : THPVariable_Wrap(std::move(q_out));
}

// cache_write(k, v, cache, device, slots) -> True
PyObject* cache_write(PyObject*, PyObject* const* a, Py_ssize_t count) {
  const chord_b200_kv_cache* cache;
  int device;
  if (count != 5 || !cache_of(a[2], a[3], &cache, &device)) return none();
  const at::Tensor *k = tensor(a[0], at::kBFloat16, 3), *v = tensor(a[1], at::kBFloat16, 3);
  if (k == nullptr || k->size(0) == 0 || !rows(k, device, k->size(0), cache->heads, cache->head_dim) ||
      !rows(v, device, k->size(0), cache->heads, cache->head_dim))
    return none();
  const int32_t* slots = ints(a[4], device, k->size(0));
  if (slots == nullptr) return none();
  int32_t* const status = devices[device].status;
  int rc;
  {
    const Unlocked unlocked;
    rc = entries.cache_write(k->const_data_ptr(), k->stride(0), k->stride(1), v->const_data_ptr(), v->stride(0), v->stride(1), cache,
                             slots, k->size(0), status, stream_of(device));
  }
  if (rc) return none();
  Py_RETURN_TRUE;
}

struct Table {
  const int32_t* at;
  int64_t stride, pages;
};

bool table_of(PyObject* o, int device, int64_t batch, Table* table) {
  const at::Tensor* t = tensor(o, at::kInt, 2);
  if (t == nullptr || t->get_device() != device || t->size(0) != batch || t->size(1) == 0 || (t->size(1) > 1 && t->stride(1) != 1) || t->stride(0) < 0)
    return false;
  *table = Table{t->const_data_ptr<int32_t>(), t->stride(0), t->size(1)};
  return true;
}

// cache_read(cache, device, block_tables, offsets, total)
PyObject* cache_read(PyObject*, PyObject* const* a, Py_ssize_t count) {
  const chord_b200_kv_cache* cache;
  int device;
  int64_t total;
  Table table;
  if (count != 5 || !cache_of(a[0], a[1], &cache, &device) || !integer(a[4], &total) || total < 1) return none();
  const at::Tensor* offsets = tensor(a[3], at::kInt, 1);
  if (offsets == nullptr || offsets->get_device() != device || offsets->size(0) < 2 || offsets->stride(0) != 1 ||
      !table_of(a[2], device, offsets->size(0) - 1, &table))
    return none();
  int32_t* const status = devices[device].status;
  at::Tensor k, v;
  int rc;
  {
    const Unlocked unlocked;
    k = empty({total, cache->heads, cache->head_dim}, *offsets), v = empty(k.sizes(), *offsets);
    rc = entries.cache_read(cache, table.at, table.stride, table.pages, offsets->const_data_ptr<int32_t>(), offsets->size(0) - 1,
                            k.mutable_data_ptr(), v.mutable_data_ptr(), total, status, stream_of(device));
  }
  return rc ? none() : pair(std::move(k), std::move(v));
}

// paged_attention(q, cache, device, block_tables, lengths, lse, window, scale)
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t count) {
  const chord_b200_kv_cache* cache;
  int device;
  int64_t window;
  double scale;
  Table table;
  if (count != 8 || !cache_of(a[1], a[2], &cache, &device) || !integer(a[6], &window) || window < 0 || window >= (1ll << 31) ||
      !number(a[7], &scale))
    return none();
  const at::Tensor* q = tensor(a[0], at::kBFloat16, 3);
  if (q == nullptr || q->size(0) == 0 || !rows(q, device, q->size(0), -1, cache->head_dim) || q->size(1) % cache->heads != 0) return none();
  const int64_t batch = q->size(0), heads = q->size(1);
  const int32_t* lengths = ints(a[4], device, batch);
  if (lengths == nullptr || !table_of(a[3], device, batch, &table)) return none();
  float* lse = nullptr;
  if (a[5] != Py_None) {
    const at::Tensor* t = tensor(a[5], at::kFloat, 2);
    if (t == nullptr || t->get_device() != device || t->size(0) != batch || t->size(1) != heads || !t->is_contiguous()) return none();
    lse = t->mutable_data_ptr<float>();
  }
  void* const stream = stream_of(device);
  int32_t* words = nullptr;
  int64_t word_count = 0;
  for (const auto& l : devices[device].locks) {
    if (l.words != nullptr && l.stream == stream) words = l.words, word_count = l.count;
  }
  const int64_t size = entries.workspace_bytes(cache->head_dim, heads / cache->heads);
  if (words == nullptr || size < 0) return none();
  int32_t* const status = devices[device].status;
  at::Tensor out;
  int rc;
  {
    const Unlocked unlocked;
    out = empty(q->sizes(), *q);
    const at::Tensor workspace = empty({size}, *q, at::kByte);
    rc = entries.paged_attention(q->const_data_ptr(), q->stride(0), q->stride(1), cache, table.at, table.stride, table.pages, lengths,
                                 out.mutable_data_ptr(), lse, words, word_count, workspace.mutable_data_ptr(), size, status, batch,
                                 heads, window, scale, stream);
  }
  return rc ? none() : THPVariable_Wrap(std::move(out));
}

// entries(addresses of the seven functions, in the struct's order)
PyObject* set_entries(PyObject*, PyObject* const* a, Py_ssize_t count) {
  int64_t at[7];
  if (count != 7) return none();
  for (int i = 0; i < 7; ++i) {
    if (!integer(a[i], at + i)) return none();
  }
  entries = {reinterpret_cast<decltype(entries.gemv)>(at[0]), reinterpret_cast<decltype(entries.qk_norm_rope)>(at[1]),
             reinterpret_cast<decltype(entries.qk_norm_rope_write)>(at[2]), reinterpret_cast<decltype(entries.cache_write)>(at[3]),
             reinterpret_cast<decltype(entries.cache_read)>(at[4]), reinterpret_cast<decltype(entries.paged_attention)>(at[5]),
             reinterpret_cast<decltype(entries.workspace_bytes)>(at[6])};
  Py_RETURN_TRUE;
}

// device(index, status word): calls may go to the device from now on.
PyObject* set_device(PyObject*, PyObject* const* a, Py_ssize_t count) {
  int64_t index, status;
  if (count != 2 || !integer(a[0], &index) || !integer(a[1], &status) || index < 0 || index >= kMaxDevices) return none();
  devices[index].status = reinterpret_cast<int32_t*>(status);
  Py_RETURN_TRUE;
}

// locks(index, stream, words, count): the default lock buffer of a stream.
PyObject* set_locks(PyObject*, PyObject* const* a, Py_ssize_t count) {
  int64_t index, stream, words, number_of;
  if (count != 4 || !integer(a[0], &index) || !integer(a[1], &stream) || !integer(a[2], &words) || !integer(a[3], &number_of) ||
      index < 0 || index >= kMaxDevices)
    return none();
  for (auto& l : devices[index].locks) {
    if (l.words != nullptr && l.stream != reinterpret_cast<void*>(stream)) continue;
    l = {reinterpret_cast<void*>(stream), reinterpret_cast<int32_t*>(words), number_of};
    Py_RETURN_TRUE;
  }
  return none();  // (further streams go through the wrapper)
}

#define METHOD(name, function) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<function>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD("gemv", gemv), METHOD("qk_norm_rope", qk_norm_rope), METHOD("qk_norm_rope_write", qk_norm_rope_write),
                         METHOD("cache_write", cache_write), METHOD("cache_read", cache_read),
                         METHOD("paged_attention", paged_attention), METHOD("entries", set_entries), METHOD("device", set_device),
                         METHOD("locks", set_locks), {nullptr, nullptr, 0, nullptr}};

// The torch whose headers this is compiled with; the package does not use it with another.
constexpr char kBuiltFor[] = "built for torch " CHORD_TORCH_VERSION;

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_call", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_call(void) {
  PyObject* const made = PyModule_Create(&module);
  if (made != nullptr && PyModule_AddStringConstant(made, "built_for", kBuiltFor) != 0) {
    Py_DECREF(made);
    return nullptr;
  }
  return made;
}
