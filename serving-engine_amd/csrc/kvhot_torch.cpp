// The per-layer calls of an engine step, from torch tensors to libkvhot's
// entry points without Python in between: paged_flash_attention, the append
// (_PagedKVCache.write) and the two together (a model's layer); and the same for
// the cache held in 4 bits, norm_rope and build_block_tables.
//
// Every function here answers the ordinary call only, after checking all that
// the Python function of the same name checks, and returns None before it has
// done anything when a check fails, when something it needs (a launch list,
// a workspace) is not there yet or when the library refuses the launch; the
// Python function then takes the call, does that preparation or raises.  (Where
// layer()'s attention is refused its append is queued already, and its answer
// says so.)  Nothing is kept between calls: pointers, shapes
// and strides are read from the tensors each time.
//
// Measured, Python with ctypes before -> here, calls queued back to back on one
// MI355X: an append of 16 tokens 8.2 -> 4.3 us, attention of one row of 1001
// keys 20.2 -> 12.1, a layer (append and attention) of 8 decode rows 33 -> 16,
// of 4 short fp32 rows 31.5 -> 12.2, 16 layers of 16 rows with their step's
// metadata and launch list 770 -> 360 to 450.  From here on the GPU's own time bounds
// all of these but the last two.
#include <Python.h>

#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/kvhot.h"
#include "../../include/kvhot_layer.h"

namespace {

using at::Tensor;

decltype(&kvhot_paged_attention) g_attention = nullptr;
decltype(&kvhot_paged_attention_workspace_bytes) g_workspace_bytes = nullptr;
decltype(&kvhot_reshape_and_cache) g_append = nullptr;
decltype(&kvhot_build_block_tables) g_tables = nullptr;
decltype(&kvhot_norm_rope) g_norm_rope = nullptr;
decltype(&kvhot_reshape_and_cache_4bit) g_append4 = nullptr;
decltype(&kvhot_read_cache_4bit) g_read4 = nullptr;
decltype(&kvhot_paged_attention_4bit_workspace_bytes) g_workspace_bytes4 = nullptr;
decltype(&kvhot_paged_attention_4bit) g_attention4 = nullptr;

// Keys of the metadata dict and of its launch lists.
struct Names {
  PyObject *q_lens, *k_lens, *q_starts, *q_pos_offsets, *block_table, *block_table_row_stride, *max_q_len, *max_k_len,
      *host_q_lens, *schedules, *schedule_streams, *total_query, *slot_mapping, *positions, *blocks_taken;
} g_names;

// The plain torch.Tensor behind o, with memory on a GPU.  (Subclasses and
// functorch's wrappers, which have no storage of their own, are not taken.)
bool gpu_tensor(PyObject* o, Tensor& t) {
  if (!o || !THPVariable_CheckExact(o)) return false;
  t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.has_storage() &&
         !t.unsafeGetTensorImpl()->key_set().has(c10::DispatchKey::Python) && !t.is_conj() && !t.is_neg();
}

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return KVHOT_F32;
    case at::kHalf: return KVHOT_F16;
    case at::kBFloat16: return KVHOT_BF16;
    default: return -1;
  }
}

// An integer that fits int64 (bool excluded: the Python path's business).
bool as_int(PyObject* o, int64_t& x) {
  if (!o || PyBool_Check(o) || !PyIndex_Check(o)) return false;
  PyObject* i = PyNumber_Index(o);
  if (!i) return false;
  int overflow = 0;
  x = PyLong_AsLongLongAndOverflow(i, &overflow);
  Py_DECREF(i);
  return overflow == 0;
}

// An int32 contiguous metadata tensor of n rows on device d.
bool meta_tensor(PyObject* meta, PyObject* name, c10::Device d, int64_t n, Tensor& t) {
  return gpu_tensor(PyDict_GetItemWithError(meta, name), t) && t.scalar_type() == at::kInt && t.device() == d &&
         t.is_contiguous() && t.dim() >= 1 && t.size(0) == n;
}

// The stream's workspace, made by the first call that needed it, if it holds
// `need` bytes; none under capture (a graph's calls have workspaces of their
// own).
bool stream_workspace(PyObject* workspaces, c10::Device d, void* stream, int64_t need, Tensor& ws) {
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(static_cast<hipStream_t>(stream), &capture) != hipSuccess) (void)hipGetLastError();
  if (capture != hipStreamCaptureStatusNone) return false;
  PyObject* key = Py_BuildValue("(iL)", static_cast<int>(d.index()),
                                static_cast<long long>(reinterpret_cast<intptr_t>(stream)));
  if (!key) return false;
  PyObject* w = PyDict_GetItemWithError(workspaces, key);
  Py_DECREF(key);
  return gpu_tensor(w, ws) && ws.numel() >= need;
}

// One layer's append: K and V new rows [1, Hkv, S, D] into the pool.
struct Append {
  Tensor kv, key, value, slots;
  int64_t layer, heads, dim;

  bool check(PyObject* kv_o, PyObject* heads_o, PyObject* dim_o, PyObject* key_o, PyObject* value_o, PyObject* layer_o,
             PyObject* slots_o) {
    if (!gpu_tensor(kv_o, kv) || !gpu_tensor(key_o, key) || !gpu_tensor(value_o, value) || !gpu_tensor(slots_o, slots) ||
        !as_int(heads_o, heads) || !as_int(dim_o, dim) || !as_int(layer_o, layer))
      return false;
    return kv.dim() == 6 && kv.size(1) == 2 && key.dim() == 4 && key.size(0) == 1 && value.sizes() == key.sizes() &&
           key.size(1) == heads && key.size(3) == dim && key.size(2) > 0 && heads > 0 && dim > 0 &&
           kv.size(4) == heads && kv.size(5) == dim && dtype_code(kv) >= 0 && key.scalar_type() == kv.scalar_type() &&
           value.scalar_type() == kv.scalar_type() && slots.dim() == 1 && slots.size(0) == key.size(2) &&
           (slots.scalar_type() == at::kLong || slots.scalar_type() == at::kInt) && slots.is_contiguous() &&
           key.device() == kv.device() && value.device() == kv.device() && slots.device() == kv.device() && layer >= 0 &&
           layer < kv.size(0);
  }
  char* pool(int64_t which) const {
    return static_cast<char*>(kv.data_ptr()) + (layer * kv.stride(0) + which * kv.stride(1)) * kv.element_size();
  }
  int launch(void* stream) const {
    const int64_t ks[3] = {key.stride(2), key.stride(1), key.stride(3)};
    const int64_t vs[3] = {value.stride(2), value.stride(1), value.stride(3)};
    const int64_t cs[4] = {kv.stride(2), kv.stride(3), kv.stride(4), kv.stride(5)};
    return g_append(key.data_ptr(), ks, value.data_ptr(), vs, pool(0), cs, pool(1), cs, slots.data_ptr(),
                    slots.scalar_type() == at::kLong ? 1 : 0, key.size(2), heads, dim, kv.size(3), kv.size(2),
                    dtype_code(kv), stream);
  }
};

// One attention call: q [T, Hq, D] over the pool's blocks.
struct Attention {
  Tensor q, k_lens, q_lens, q_starts, q_offs, bt, units, ws;
  const void *k = nullptr, *v = nullptr;
  int64_t kst[4], vst[4], num_blocks, block_size, hkv;
  int64_t bt_stride, max_q, max_k, counts[4], need, pt;
  bool listed = false;
  float scale;
  int flags;
  void* stream;

  // Whether the stream comes after the copy of the launch list of `key`
  // (_order_list's record; a list without one is taken as it is).
  bool list_ordered(PyObject* meta, PyObject* key) const {
    PyObject* all = PyDict_GetItemWithError(meta, g_names.schedule_streams);
    PyObject* rec = all && PyDict_CheckExact(all) ? PyDict_GetItemWithError(all, key) : nullptr;
    if (!rec) return !PyErr_Occurred();
    if (!PyTuple_CheckExact(rec) || PyTuple_GET_SIZE(rec) != 2 || !PySet_Check(PyTuple_GET_ITEM(rec, 1))) return false;
    PyObject* h = PyLong_FromLongLong(static_cast<long long>(reinterpret_cast<intptr_t>(stream)));
    if (!h) return false;
    const int in = PySet_Contains(PyTuple_GET_ITEM(rec, 1), h);
    Py_DECREF(h);
    return in == 1;
  }

  // q, the pool and hkv are set; the rest from the metadata.
  bool check(PyObject* meta, PyObject* scale_o, int64_t pt_, bool causal, int flags_, PyObject* workspaces) {
    if (!PyDict_CheckExact(meta) || !PyDict_CheckExact(workspaces) || !PyFloat_Check(scale_o)) return false;
    scale = static_cast<float>(PyFloat_AS_DOUBLE(scale_o));
    pt = pt_;
    flags = flags_;
    const c10::Device d = q.device();
    const int64_t hq = q.size(1), dim = q.size(2);
    stream = c10::hip::getCurrentHIPStream(d.index()).stream();
    const int dt = dtype_code(q);
    if (dt < 0 || hkv <= 0 || hq <= 0 || hq % hkv != 0 || q.size(0) == 0 || dim == 0) return false;
    if (!gpu_tensor(PyDict_GetItemWithError(meta, g_names.q_lens), q_lens) || q_lens.dim() < 1) return false;
    const int64_t rows = q_lens.size(0);
    if (rows == 0 || q_lens.scalar_type() != at::kInt || q_lens.device() != d || !q_lens.is_contiguous() ||
        !meta_tensor(meta, g_names.k_lens, d, rows, k_lens) || !meta_tensor(meta, g_names.q_starts, d, rows, q_starts) ||
        !meta_tensor(meta, g_names.q_pos_offsets, d, rows, q_offs) || !meta_tensor(meta, g_names.block_table, d, rows, bt))
      return false;
    PyObject* st = PyDict_GetItemWithError(meta, g_names.block_table_row_stride);
    if (st) {
      if (!as_int(st, bt_stride)) return false;
    } else {
      bt_stride = bt.dim() == 2 ? bt.size(1) : 0;
    }
    if (!as_int(PyDict_GetItemWithError(meta, g_names.max_q_len), max_q) ||
        !as_int(PyDict_GetItemWithError(meta, g_names.max_k_len), max_k))
      return false;
    PyObject* host = PyDict_GetItemWithError(meta, g_names.host_q_lens);
    if (host && host != Py_None) {
      // The step's launch list, built by the first call of its shape.
      PyObject* lists = PyDict_GetItemWithError(meta, g_names.schedules);
      if (!lists || !PyDict_CheckExact(lists)) return false;
      char name[16];
      snprintf(name, sizeof name, "cuda:%d", static_cast<int>(d.index()));
      PyObject* key = Py_BuildValue("(LLLLLOis)", (long long)hq, (long long)hkv, (long long)dim, (long long)block_size,
                                    (long long)pt, causal ? Py_True : Py_False, dt, name);
      if (!key) return false;
      PyObject* hit = PyDict_GetItemWithError(lists, key);
      const bool ordered = hit && (hit == Py_None || list_ordered(meta, key));
      Py_DECREF(key);
      if (!ordered) return false;
      if (hit != Py_None) {
        if (!PyTuple_CheckExact(hit) || PyTuple_GET_SIZE(hit) != 6) return false;
        // (device units, decode, prefill, merge units, workspace bytes, prefix units)
        if (!as_int(PyTuple_GET_ITEM(hit, 1), counts[0]) || !as_int(PyTuple_GET_ITEM(hit, 2), counts[1]) ||
            !as_int(PyTuple_GET_ITEM(hit, 3), counts[2]) || !as_int(PyTuple_GET_ITEM(hit, 4), need) ||
            !as_int(PyTuple_GET_ITEM(hit, 5), counts[3]) || !gpu_tensor(PyTuple_GET_ITEM(hit, 0), units))
          return false;
        listed = counts[0] + counts[1] > 0;
      }
    }
    if (!listed) {
      counts[0] = counts[1] = counts[2] = counts[3] = 0;
      need = g_workspace_bytes(rows, q.size(0), max_q, max_k, hq, hkv, dim, block_size, pt, dt);
      if (need < 0) return false;
    }
    return need == 0 || stream_workspace(workspaces, d, stream, need, ws);
  }

  int launch(const Tensor& o, const Tensor& l) const {
    const int64_t qs[3] = {q.stride(0), q.stride(1), q.stride(2)}, os[3] = {o.stride(0), o.stride(1), o.stride(2)};
    const int64_t ls[2] = {l.stride(0), l.stride(1)};
    const auto i32 = [](const Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); };
    return g_attention(q.data_ptr(), qs, k, kst, v, vst, o.data_ptr(), os, static_cast<float*>(l.data_ptr()), ls, i32(bt),
                       bt_stride, i32(q_lens), i32(k_lens), i32(q_starts), i32(q_offs), q_lens.size(0), q.size(0), max_q,
                       max_k, q.size(1), hkv, q.size(2), block_size, num_blocks, scale, flags, dtype_code(q), pt,
                       listed ? i32(units) : nullptr, counts[0], counts[1], counts[2], counts[3], listed ? need : 0,
                       ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? ws.numel() : 0, stream);
  }
};

// The call's Python result, or None with no error set.
template <class F>
PyObject* or_none(F f) {
  PyObject* r = nullptr;
  try {
    r = f();
  } catch (...) {
    r = nullptr;
  }
  if (!r) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  return r;
}

// f() without the GIL, which is taken again whichever way f ends.
template <class F>
int without_gil(F f) {
  struct Released {
    PyThreadState* state = PyEval_SaveThread();
    ~Released() { PyEval_RestoreThread(state); }
  } released;
  return f();
}

Tensor lse_of(const Tensor& q) {
  return at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat).requires_grad(false).memory_format(c10::nullopt));
}

PyObject* pair_of(const Tensor& x, const Tensor& y) {
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(x));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(y));
  return r;
}

// attention(q, k_cache, v_cache, metadata, hq, hkv, scale, causal, pt, flags, workspaces) -> (o, l) | None
PyObject* py_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return or_none([&]() -> PyObject* {
    Tensor k, v;
    Attention at_;
    int64_t hq, pt, flags;
    if (n != 11 || !g_attention || !gpu_tensor(a[0], at_.q) || !gpu_tensor(a[1], k) || !gpu_tensor(a[2], v) ||
        !as_int(a[4], hq) || !as_int(a[5], at_.hkv) || !as_int(a[8], pt) || !as_int(a[9], flags) || !PyBool_Check(a[7]))
      return nullptr;
    const Tensor& q = at_.q;
    if (q.dim() != 3 || k.dim() != 4 || v.sizes() != k.sizes() || q.size(1) != hq || k.size(2) != at_.hkv ||
        k.size(3) != q.size(2) || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() ||
        k.device() != q.device() || v.device() != q.device())
      return nullptr;
    for (int i = 0; i < 4; ++i) {
      at_.kst[i] = k.stride(i);
      at_.vst[i] = v.stride(i);
    }
    at_.k = k.data_ptr();
    at_.v = v.data_ptr();
    at_.num_blocks = k.size(0);
    at_.block_size = k.size(1);
    if (!at_.check(a[3], a[6], pt, a[7] == Py_True, static_cast<int>(flags), a[10])) return nullptr;
    const Tensor o = at::empty_like(q, q.options().requires_grad(false)), l = lse_of(q);
    if (without_gil([&] { return at_.launch(o, l); }) != 0) return nullptr;
    return pair_of(o, l);
  });
}

// append(kv_cache, heads, dim, key, value, layer, slots) -> True | None
PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return or_none([&]() -> PyObject* {
    Append ap;
    if (n != 7 || !g_append || !ap.check(a[0], a[1], a[2], a[3], a[4], a[5], a[6])) return nullptr;
    void* stream = c10::hip::getCurrentHIPStream(ap.kv.device().index()).stream();
    if (without_gil([&] { return ap.launch(stream); }) != 0) return nullptr;
    Py_RETURN_TRUE;
  });
}

// layer(kv_cache, heads, dim, key, value, layer, slots, query, metadata, scale, pt, flags, workspaces)
//   -> o [1, S, Hq, D] | None | False: the append, then causal attention; False
//   where the append is queued and the library then refused the attention.
PyObject* py_layer(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return or_none([&]() -> PyObject* {
    Append ap;
    Attention at_;
    Tensor query;
    int64_t pt, flags;
    if (n != 13 || !g_append || !g_attention || !ap.check(a[0], a[1], a[2], a[3], a[4], a[5], a[6]) ||
        !gpu_tensor(a[7], query) || !as_int(a[10], pt) || !as_int(a[11], flags))
      return nullptr;
    const Tensor& kv = ap.kv;
    if (query.dim() != 4 || query.size(0) != 1 || query.size(3) != ap.dim ||
        query.scalar_type() != kv.scalar_type() || query.device() != kv.device())
      return nullptr;
    at_.q = query.transpose(1, 2).squeeze(0);
    if (at_.q.dim() != 3) return nullptr;
    for (int i = 0; i < 4; ++i) at_.kst[i] = at_.vst[i] = kv.stride(2 + i);
    at_.k = ap.pool(0);
    at_.v = ap.pool(1);
    at_.num_blocks = kv.size(2);
    at_.block_size = kv.size(3);
    at_.hkv = ap.heads;
    if (!at_.check(a[8], a[9], pt, true, static_cast<int>(flags), a[12])) return nullptr;
    const Tensor o = at::empty_like(at_.q, at_.q.options().requires_grad(false)), l = lse_of(at_.q);
    if (without_gil([&] { return ap.launch(at_.stream); }) != 0) return nullptr;
    // (An exception here, from a library call that could not form its message,
    // is such a refusal too.)
    int status = -1;
    try {
      status = without_gil([&] { return at_.launch(o, l); });
    } catch (...) {
    }
    if (status != 0) Py_RETURN_FALSE;
    return THPVariable_Wrap(o.unsqueeze(0));
  });
}

// ------------------------------------------------------- include/kvhot_layer.h

// Whether t's device is the current one (the Python functions switch to it).
bool on_current_device(const Tensor& t) {
  int now = -1;
  return hipGetDevice(&now) == hipSuccess && now == t.get_device();
}

bool index_tensor(const Tensor& t, c10::Device d) {
  return t.dim() == 1 && (t.scalar_type() == at::kLong || t.scalar_type() == at::kInt) && t.is_contiguous() &&
         t.device() == d;
}

bool is_long(const Tensor& t) { return t.scalar_type() == at::kLong; }

// A layer of a cache held in 4 bits: records [N, S, Hkv, 17 D].
struct Pool4Bit {
  Tensor pool;  // [L, N, S, Hkv, 17 D]
  int64_t layer, dim;

  bool check(PyObject* pool_o, PyObject* dim_o, PyObject* layer_o) {
    return gpu_tensor(pool_o, pool) && as_int(dim_o, dim) && as_int(layer_o, layer) && pool.dim() == 5 &&
           pool.scalar_type() == at::kByte && layer >= 0 && layer < pool.size(0) && pool.size(4) == 17 * dim &&
           pool.stride(4) == 1 && pool.stride(3) == 17 * dim && pool.stride(2) == pool.size(3) * 17 * dim &&
           on_current_device(pool);
  }
  char* base() const { return static_cast<char*>(pool.data_ptr()) + layer * pool.stride(0); }
  int64_t heads() const { return pool.size(3); }
  int64_t block_size() const { return pool.size(2) * 16; }
};

// append4(pool, dim, dtype, key, value, layer, slots) -> True | None
PyObject* py_append4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return or_none([&]() -> PyObject* {
    Pool4Bit p;
    Tensor key, value, slots;
    int64_t dtype;
    if (n != 7 || !g_append4 || !p.check(a[0], a[1], a[5]) || !as_int(a[2], dtype) || !gpu_tensor(a[3], key) ||
        !gpu_tensor(a[4], value) || !gpu_tensor(a[6], slots))
      return nullptr;
    const c10::Device d = p.pool.device();
    if (key.dim() != 4 || key.size(0) != 1 || value.sizes() != key.sizes() || key.size(1) != p.heads() ||
        key.size(3) != p.dim || key.size(2) == 0 || dtype_code(key) != dtype || dtype_code(value) != dtype ||
        key.device() != d || value.device() != d || !index_tensor(slots, d) || slots.size(0) != key.size(2))
      return nullptr;
    const int64_t ks[3] = {key.stride(2), key.stride(1), key.stride(3)};
    const int64_t vs[3] = {value.stride(2), value.stride(1), value.stride(3)};
    void* stream = c10::hip::getCurrentHIPStream(d.index()).stream();
    const int status = without_gil([&] {
      return g_append4(key.data_ptr(), ks, value.data_ptr(), vs, p.base(), p.pool.stride(1), slots.data_ptr(),
                       is_long(slots), key.size(2), p.heads(), p.dim, p.block_size(), p.pool.size(1),
                       static_cast<int>(dtype), stream);
    });
    if (status != 0) return nullptr;
    Py_RETURN_TRUE;
  });
}

// read4(pool, dim, dtype, layer, slots) -> (key, value) | None
PyObject* py_read4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return or_none([&]() -> PyObject* {
    Pool4Bit p;
    Tensor slots;
    int64_t dtype;
    if (n != 5 || !g_read4 || !p.check(a[0], a[1], a[3]) || !as_int(a[2], dtype) || !gpu_tensor(a[4], slots) ||
        !index_tensor(slots, p.pool.device()) || slots.size(0) == 0)
      return nullptr;
    const at::ScalarType type = dtype == KVHOT_F32 ? at::kFloat : dtype == KVHOT_F16 ? at::kHalf : at::kBFloat16;
    const auto options = p.pool.options().dtype(type);
    const at::AutoDispatchBelowADInplaceOrView plain;  // (no gradients here: new tensors and views of them)
    const Tensor key = at::empty({slots.size(0), p.heads(), p.dim}, options), value = at::empty(key.sizes(), options);
    void* stream = c10::hip::getCurrentHIPStream(p.pool.get_device()).stream();
    const int status = without_gil([&] {
      return g_read4(p.base(), p.pool.stride(1), slots.data_ptr(), is_long(slots), slots.size(0), p.heads(), p.dim,
                     p.block_size(), p.pool.size(1), key.data_ptr(), value.data_ptr(), 0, static_cast<int>(dtype), stream);
    });
    if (status != 0) return nullptr;
    return pair_of(key, value);
  });
}

// attention4(q, blocks, metadata, hq, hkv, scale, causal, workspaces, prompt_pairs) -> (o, l) | None
//   (None where the host knows of a row that may have that many (query, head) pairs
//   a kv head, unless the step's plan is there and has no prompts.)
PyObject* py_attention4(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return or_none([&]() -> PyObject* {
    Tensor q, kv, q_lens, k_lens, q_starts, q_offs, bt, ws;
    int64_t hq, hkv, max_q, max_k, bt_stride, prompt;
    if (n != 9 || !as_int(a[8], prompt) || !g_attention4 || !g_workspace_bytes4 || !gpu_tensor(a[0], q) || !gpu_tensor(a[1], kv) ||
        !PyDict_CheckExact(a[2]) || !as_int(a[3], hq) || !as_int(a[4], hkv) || !PyFloat_Check(a[5]) || !PyBool_Check(a[6]) ||
        !PyDict_CheckExact(a[7]))
      return nullptr;
    PyObject* meta = a[2];
    const int dt = dtype_code(q);
    const c10::Device d = q.device();
    if (q.dim() != 3 || kv.dim() != 4 || kv.scalar_type() != at::kByte || kv.device() != d || dt < 0 || hkv <= 0 || hq <= 0 ||
        hq % hkv != 0 || q.size(1) != hq || q.size(0) == 0 || kv.size(2) != hkv || kv.size(3) != 17 * q.size(2) ||
        kv.stride(3) != 1 || kv.stride(2) != kv.size(3) || kv.stride(1) != hkv * kv.size(3) || !on_current_device(q))
      return nullptr;
    if (!gpu_tensor(PyDict_GetItemWithError(meta, g_names.q_lens), q_lens) || q_lens.dim() < 1) return nullptr;
    const int64_t rows = q_lens.size(0);
    if (rows == 0 || !meta_tensor(meta, g_names.q_lens, d, rows, q_lens) || !meta_tensor(meta, g_names.k_lens, d, rows, k_lens) ||
        !meta_tensor(meta, g_names.q_starts, d, rows, q_starts) || !meta_tensor(meta, g_names.q_pos_offsets, d, rows, q_offs) ||
        !meta_tensor(meta, g_names.block_table, d, rows, bt) ||
        !as_int(PyDict_GetItemWithError(meta, g_names.block_table_row_stride), bt_stride) ||
        !as_int(PyDict_GetItemWithError(meta, g_names.max_q_len), max_q) ||
        !as_int(PyDict_GetItemWithError(meta, g_names.max_k_len), max_k))
      return nullptr;
    PyObject* host = PyDict_GetItemWithError(meta, g_names.host_q_lens);
    if (host && host != Py_None && dt != KVHOT_F32 && hq / hkv <= 16 && max_q * (hq / hkv) >= prompt) {
      PyObject* plans = PyDict_GetItemWithError(meta, g_names.schedules);
      if (!plans || !PyDict_CheckExact(plans)) return nullptr;
      char name[16];
      snprintf(name, sizeof name, "cuda:%d", static_cast<int>(d.index()));
      PyObject* key = Py_BuildValue("(sLLLLis)", "prompts4", (long long)hq, (long long)hkv, (long long)q.size(2),
                                    (long long)(kv.size(1) * 16), dt, name);
      if (!key) return nullptr;
      PyObject* hit = PyDict_GetItemWithError(plans, key);
      Py_DECREF(key);
      if (hit != Py_None) return nullptr;
    }
    const int64_t need = g_workspace_bytes4(rows, q.size(0), max_q, max_k, hq, hkv, q.size(2), dt);
    void* stream = c10::hip::getCurrentHIPStream(d.index()).stream();
    if (need < 0 || (need > 0 && !stream_workspace(a[7], d, stream, need, ws))) return nullptr;
    const at::AutoDispatchBelowADInplaceOrView plain;
    const Tensor o = at::empty_like(q, q.options().requires_grad(false)), l = lse_of(q);
    const int64_t qs[3] = {q.stride(0), q.stride(1), q.stride(2)}, os[3] = {o.stride(0), o.stride(1), o.stride(2)};
    const int64_t ls[2] = {l.stride(0), l.stride(1)};
    const float scale = static_cast<float>(PyFloat_AS_DOUBLE(a[5]));
    const int flags = a[6] == Py_True ? KVHOT_CAUSAL : 0;
    const auto i32 = [](const Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); };
    const int status = without_gil([&] {
      return g_attention4(q.data_ptr(), qs, kv.data_ptr(), kv.stride(0), o.data_ptr(), os, static_cast<float*>(l.data_ptr()),
                          ls, i32(bt), bt_stride, i32(q_lens), i32(k_lens), i32(q_starts), i32(q_offs), rows, q.size(0), q.size(0),
                          max_q, max_k, hq, hkv, q.size(2), kv.size(1) * 16, kv.size(0), scale, flags, dt,
                          ws.defined() ? ws.data_ptr() : nullptr, ws.defined() ? ws.numel() : 0, stream);
    });
    if (status != 0) return nullptr;
    return pair_of(o, l);
  });
}

// norm_rope(q, k, positions, table, q_weight, k_weight, eps, interleaved) -> (q', k') | None
PyObject* py_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return or_none([&]() -> PyObject* {
    Tensor q, k, pos, table, w[2];
    if (n != 8 || !g_norm_rope || !gpu_tensor(a[0], q) || !gpu_tensor(a[1], k) || !gpu_tensor(a[2], pos) ||
        !gpu_tensor(a[3], table) || !PyFloat_Check(a[6]) || !PyBool_Check(a[7]))
      return nullptr;
    const int dt = dtype_code(q);
    const c10::Device d = q.device();
    if (q.dim() != 3 || k.dim() != 3 || dt < 0 || k.scalar_type() != q.scalar_type() || q.size(0) != k.size(0) ||
        q.size(2) != k.size(2) || q.size(0) == 0 || k.device() != d || !index_tensor(pos, d) || pos.size(0) != q.size(0) ||
        table.dim() != 2 || table.scalar_type() != at::kFloat || !table.is_contiguous() || table.device() != d ||
        !on_current_device(q))
      return nullptr;
    int wdt = dt;
    for (int i = 0; i < 2; ++i) {
      if (a[4 + i] == Py_None) continue;
      if (!gpu_tensor(a[4 + i], w[i]) || w[i].dim() != 1 || w[i].size(0) != q.size(2) || !w[i].is_contiguous() ||
          w[i].device() != d || (w[i].scalar_type() != at::kFloat && w[i].scalar_type() != q.scalar_type()) ||
          (i == 1 && w[0].defined() && w[0].scalar_type() != w[1].scalar_type()))
        return nullptr;
      wdt = dtype_code(w[i]);
    }
    const auto options = q.options().requires_grad(false);
    const at::AutoDispatchBelowADInplaceOrView plain;
    const Tensor oq = at::empty(q.sizes(), options), ok = at::empty(k.sizes(), options);
    const Tensor* t[4] = {&q, &k, &oq, &ok};
    int64_t st[4][3];
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 3; ++j) st[i][j] = t[i]->stride(j);
    const auto weight = [&](int i) { return w[i].defined() ? w[i].data_ptr() : nullptr; };
    const float eps = static_cast<float>(PyFloat_AS_DOUBLE(a[6]));
    const int interleaved = a[7] == Py_True ? 1 : 0;
    void* stream = c10::hip::getCurrentHIPStream(d.index()).stream();
    const int status = without_gil([&] {
      return g_norm_rope(q.data_ptr(), st[0], k.data_ptr(), st[1], oq.data_ptr(), st[2], ok.data_ptr(), st[3], weight(0),
                         weight(1), wdt, eps, static_cast<const float*>(table.data_ptr()), table.size(0), table.size(1),
                         interleaved, pos.data_ptr(), is_long(pos), q.size(0), q.size(1), k.size(1), q.size(2), dt, stream);
    });
    if (status != 0) return nullptr;
    return pair_of(oq, ok);
  });
}

// tables(block_table, prior_lens, q_lens, free_blocks, total, max_q, max_k, block_size) -> metadata dict | None
PyObject* py_tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return or_none([&]() -> PyObject* {
    Tensor bt, prior, q_lens, free;
    int64_t total, max_q, max_k, bs;
    if (n != 8 || !g_tables || !gpu_tensor(a[0], bt) || !gpu_tensor(a[1], prior) || !gpu_tensor(a[2], q_lens) ||
        !gpu_tensor(a[3], free) || !as_int(a[4], total) || !as_int(a[5], max_q) || !as_int(a[6], max_k) || !as_int(a[7], bs))
      return nullptr;
    const c10::Device d = bt.device();
    const auto list = [&](const Tensor& t) {
      return t.dim() == 1 && t.scalar_type() == at::kInt && t.is_contiguous() && t.device() == d;
    };
    if (bt.dim() != 2 || bt.scalar_type() != at::kInt || !bt.is_contiguous() || !list(prior) || !list(q_lens) || !list(free) ||
        prior.size(0) != bt.size(0) || q_lens.size(0) != bt.size(0) || bt.size(0) == 0 || total < 0 || max_q < 0 || bs <= 0 ||
        !on_current_device(bt))
      return nullptr;
    const int64_t r = bt.size(0), mb = bt.size(1);
    const at::AutoDispatchBelowADInplaceOrView plain;
    const Tensor ints = at::empty({2 * r + 1}, bt.options()), longs = at::empty({2 * total}, bt.options().dtype(at::kLong));
    int32_t* const i = static_cast<int32_t*>(ints.data_ptr());
    int64_t* const l = static_cast<int64_t*>(longs.data_ptr());
    const auto i32 = [](const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); };
    void* stream = c10::hip::getCurrentHIPStream(d.index()).stream();
    const int status = without_gil([&] {
      return g_tables(i32(bt), mb, i32(prior), i32(q_lens), i32(free), free.size(0), r, total, max_q, bs, i + r, i, l,
                      l + total, i + 2 * r, stream);
    });
    if (status != 0) return nullptr;
    PyObject* meta = PyDict_New();
    if (!meta) return nullptr;
    const auto put = [&](PyObject* name, PyObject* x) {  // takes x
      const bool ok = x && PyDict_SetItem(meta, name, x) == 0;
      Py_XDECREF(x);
      return ok;
    };
    bool ok = true;
    try {
      ok = put(g_names.q_lens, Py_NewRef(a[2])) && put(g_names.k_lens, THPVariable_Wrap(ints.narrow(0, 0, r))) &&
           put(g_names.q_starts, THPVariable_Wrap(ints.narrow(0, r, r))) && put(g_names.q_pos_offsets, Py_NewRef(a[1])) &&
           put(g_names.block_table, Py_NewRef(a[0])) && put(g_names.block_table_row_stride, PyLong_FromLongLong(mb)) &&
           put(g_names.total_query, PyLong_FromLongLong(total)) && put(g_names.max_q_len, PyLong_FromLongLong(max_q)) &&
           put(g_names.max_k_len, PyLong_FromLongLong(max_k)) &&
           put(g_names.slot_mapping, THPVariable_Wrap(longs.narrow(0, 0, total))) &&
           put(g_names.positions, THPVariable_Wrap(longs.narrow(0, total, total))) &&
           put(g_names.blocks_taken, THPVariable_Wrap(ints.narrow(0, 2 * r, 1)));
    } catch (...) {
      ok = false;
    }
    if (!ok) {
      Py_DECREF(meta);
      return nullptr;
    }
    return meta;
  });
}

// bind_layer(addresses of kvhot_layer.h's entry points, in its order)
PyObject* py_bind_layer(PyObject*, PyObject* args) {
  unsigned long long f[6];
  if (!PyArg_ParseTuple(args, "KKKKKK", f, f + 1, f + 2, f + 3, f + 4, f + 5)) return nullptr;
  const auto at = [&](int i) { return static_cast<uintptr_t>(f[i]); };
  g_tables = reinterpret_cast<decltype(g_tables)>(at(0));
  g_norm_rope = reinterpret_cast<decltype(g_norm_rope)>(at(1));
  g_append4 = reinterpret_cast<decltype(g_append4)>(at(2));
  g_read4 = reinterpret_cast<decltype(g_read4)>(at(3));
  g_workspace_bytes4 = reinterpret_cast<decltype(g_workspace_bytes4)>(at(4));
  g_attention4 = reinterpret_cast<decltype(g_attention4)>(at(5));
  Py_RETURN_NONE;
}

// bind(attention, workspace_bytes, append): addresses of libkvhot's entry points.
PyObject* py_bind(PyObject*, PyObject* args) {
  unsigned long long at, ws, ap;
  if (!PyArg_ParseTuple(args, "KKK", &at, &ws, &ap)) return nullptr;
  g_attention = reinterpret_cast<decltype(g_attention)>(static_cast<uintptr_t>(at));
  g_workspace_bytes = reinterpret_cast<decltype(g_workspace_bytes)>(static_cast<uintptr_t>(ws));
  g_append = reinterpret_cast<decltype(g_append)>(static_cast<uintptr_t>(ap));
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_attention)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_append)), METH_FASTCALL, nullptr},
    {"layer", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_layer)), METH_FASTCALL, nullptr},
    {"bind", py_bind, METH_VARARGS, nullptr},
    {"append4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_append4)), METH_FASTCALL, nullptr},
    {"read4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_read4)), METH_FASTCALL, nullptr},
    {"attention4", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_attention4)), METH_FASTCALL, nullptr},
    {"norm_rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_norm_rope)), METH_FASTCALL, nullptr},
    {"tables", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_tables)), METH_FASTCALL, nullptr},
    {"bind_layer", py_bind_layer, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "kvhot_torch", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_kvhot_torch(void) {
  Names& g = g_names;
  g.q_lens = PyUnicode_InternFromString("q_lens");
  g.k_lens = PyUnicode_InternFromString("k_lens");
  g.q_starts = PyUnicode_InternFromString("q_starts");
  g.q_pos_offsets = PyUnicode_InternFromString("q_pos_offsets");
  g.block_table = PyUnicode_InternFromString("block_table");
  g.block_table_row_stride = PyUnicode_InternFromString("block_table_row_stride");
  g.max_q_len = PyUnicode_InternFromString("max_q_len");
  g.max_k_len = PyUnicode_InternFromString("max_k_len");
  g.host_q_lens = PyUnicode_InternFromString("host_q_lens");
  g.schedules = PyUnicode_InternFromString("_schedules");
  g.schedule_streams = PyUnicode_InternFromString("_schedule_streams");
  g.total_query = PyUnicode_InternFromString("total_query");
  g.slot_mapping = PyUnicode_InternFromString("slot_mapping");
  g.positions = PyUnicode_InternFromString("positions");
  g.blocks_taken = PyUnicode_InternFromString("blocks_taken");
  return PyModule_Create(&kModule);
}
