// Host side of the short calls, compiled: paged decode of a batch, the KV
// gather and a serving step's operators take microseconds on the device, and reading a dozen tensors'
// properties from Python took longer than that (5 x 1000 tokens, 8 x 96
// float32, two launches: 17.7 -> 9.4 us a call; 1 x 2048 bfloat16 with the
// append 18.9 -> 9.5 us; twelve layers of append and gather at 8192 tokens 188
// -> 152 us; reserve of 64 rows 16.5 -> 9.4 us, rope_append of 64 tokens 15.6 ->
// 5.1).  Each function here takes the tensors,
// checks the form the usual calls have, allocates the results and queues the
// launches through the library's C entry points; for any other form it returns
// None and the caller goes through the checks written in Python, which raise
// what is wrong.  A failed entry point's status is returned as an int.
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "mie_paged_kv.h"

namespace {

// The entry points, from the library the process has already loaded.
decltype(&mie_paged_decode) g_decode;
decltype(&mie_paged_decode_append) g_decode_append;
decltype(&mie_paged_decode_plan) g_plan;
decltype(&mie_paged_decode_plan_known) g_plan_known;
decltype(&mie_kv_gather) g_gather;
decltype(&mie_step_reserve) g_reserve;
decltype(&mie_step_release) g_release;
decltype(&mie_rope_append) g_rope;
decltype(&mie_paged_extend_workspace) g_extend_workspace;
decltype(&mie_paged_extend) g_extend;
decltype(&mie_token_logprobs_workspace) g_logprobs_workspace;
decltype(&mie_token_logprobs) g_logprobs;

// A plain ROCm tensor: no subclass, no functorch or dispatch wrapper, storage
// of its own device.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided || t.is_neg() || t.is_conj()) return nullptr;
  const auto keys = t.key_set();
  if (keys.has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched,
                                        c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::BatchedNestedTensor,
                                        c10::DispatchKey::Functionalize})))
    return nullptr;
  return &t;
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return MIE_DTYPE_F32;
    case at::kBFloat16: return MIE_DTYPE_BF16;
    default: return -1;
  }
}

bool as_int(PyObject* o, int64_t& out) {
  if (!PyLong_CheckExact(o)) return false;
  out = PyLong_AsLongLong(o);
  if (out == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

bool fits(int64_t v) { return v >= 0 && v <= INT32_MAX; }

// decode(q, k_pool, v_pool, layer, tables, lens, max_len, host_lens, scale,
//        partition, k_new, v_new, stream) -> out, None or a status
// q [B, H, D], pools [L, NB, H, BS, D], tables int32 [B, n], lens int32 [B];
// host_lens a list of ints or None; scale a float or None; k_new, v_new
// [B, H, D] or None.
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13) Py_RETURN_NONE;
  const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]), *tables = plain(a[4]), *lens = plain(a[5]);
  int64_t layer, max_len, partition, stream;
  if (!q || !k || !v || !tables || !lens || !as_int(a[3], layer) || !as_int(a[6], max_len) ||
      !as_int(a[9], partition) || !as_int(a[12], stream))
    Py_RETURN_NONE;
  if (q->dim() != 3 || k->dim() != 5 || tables->dim() != 2 || lens->dim() != 1) Py_RETURN_NONE;
  const auto qs = q->sizes(), ks = k->sizes();
  const auto qt = q->strides(), kt = k->strides();
  const int code = dtype_code(q->scalar_type());
  const auto device = q->device();
  const int64_t batch = qs[0], heads = qs[1], dim = qs[2], blocks = ks[1], block = ks[3];
  if (code < 0 || k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() ||
      k->device() != device || v->device() != device || tables->device() != device || lens->device() != device ||
      tables->scalar_type() != at::kInt || lens->scalar_type() != at::kInt || v->sizes() != ks || v->strides() != kt ||
      layer < 0 || layer >= ks[0] || ks[2] != heads || ks[4] != dim || kt[4] != 1 || kt[3] != dim || qt[2] != 1 ||
      tables->size(0) != batch || tables->stride(1) != 1 || lens->size(0) != batch || !lens->is_contiguous() ||
      !fits(batch) || !fits(heads) || !fits(blocks) || !fits(block) || !fits(max_len) || partition < -1 ||
      partition > INT32_MAX)
    Py_RETURN_NONE;
  double scale = 1.0 / std::sqrt(static_cast<double>(dim));
  if (a[8] != Py_None) {
    if (!PyFloat_CheckExact(a[8])) Py_RETURN_NONE;
    scale = PyFloat_AS_DOUBLE(a[8]);
  }
  std::vector<int32_t> host;
  int64_t longest = 0;
  if (a[7] != Py_None) {
    if (!PyList_CheckExact(a[7]) || PyList_GET_SIZE(a[7]) != batch) Py_RETURN_NONE;
    host.resize(batch);
    for (int64_t b = 0; b < batch; ++b) {
      int64_t c;
      if (!as_int(PyList_GET_ITEM(a[7], b), c) || c < INT32_MIN || c > INT32_MAX) Py_RETURN_NONE;
      host[b] = static_cast<int32_t>(c);
      longest = std::max(longest, std::min(c, max_len));
    }
  }
  const at::Tensor *kn = nullptr, *vn = nullptr;
  if (a[10] != Py_None || a[11] != Py_None) {
    kn = plain(a[10]);
    vn = plain(a[11]);
    for (const at::Tensor* t : {kn, vn})
      if (!t || t->sizes() != qs || t->scalar_type() != q->scalar_type() || t->device() != device || t->stride(2) != 1)
        Py_RETURN_NONE;
    if (kn->strides() != vn->strides()) Py_RETURN_NONE;
  }
  int32_t part = static_cast<int32_t>(partition);
  int64_t bytes = 0;
  int32_t rc = a[7] != Py_None && partition == 0
                   ? g_plan_known(batch, heads, dim, block, max_len, longest, kn != nullptr, code, &part, &bytes)
                   : g_plan(batch, heads, dim, block, max_len, code, partition, nullptr, &bytes);
  if (rc != MIE_OK) return PyLong_FromLong(rc);
  at::Tensor out = at::empty({batch, heads, dim}, q->options().requires_grad(false));
  at::Tensor ws;
  if (bytes > 0) ws = at::empty({bytes}, q->options().dtype(at::kByte).requires_grad(false));
  const int64_t offset = layer * kt[0] * q->element_size();
  char* kp = static_cast<char*>(k->data_ptr()) + offset;
  char* vp = static_cast<char*>(v->data_ptr()) + offset;
  const int32_t* tab = static_cast<const int32_t*>(tables->data_ptr());
  const int32_t* len = static_cast<const int32_t*>(lens->data_ptr());
  const int32_t* hl = host.empty() ? nullptr : host.data();
  void* wsp = bytes > 0 ? ws.data_ptr() : nullptr;
  void* st = reinterpret_cast<void*>(stream);
  void* op = out.data_ptr();
  const void* qp = q->data_ptr();
  const void* knp = kn ? kn->data_ptr() : nullptr;
  const void* vnp = vn ? vn->data_ptr() : nullptr;
  const int64_t nb = kn ? kn->stride(0) : 0, nh = kn ? kn->stride(1) : 0, ts = tables->stride(0);
  // A launch waits when the queue is full: not with the interpreter held.
  Py_BEGIN_ALLOW_THREADS
  if (kn) {
    rc = g_decode_append(qp, qt[0], qt[1], kp, vp, kt[1], kt[2], blocks, tab, ts, len, hl, 0, max_len, batch, heads,
                         dim, block, static_cast<float>(scale), op, heads * dim, dim, code, wsp, bytes, part, knp,
                         vnp, nb, nh, code, st);
  } else {
    rc = g_decode(qp, qt[0], qt[1], kp, vp, kt[1], kt[2], blocks, tab, ts, len, hl, 0, max_len, batch, heads, dim,
                  block, static_cast<float>(scale), op, heads * dim, dim, code, wsp, bytes, part, code, st);
  }
  Py_END_ALLOW_THREADS
  if (rc != MIE_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// gather(k_pool, v_pool, layer, table, length, stream) -> (K, V), None or a status
// Contiguous pools [L, NB, H, BS, D] of one dtype, table int32 with an entry
// per block of the pool.
PyObject* gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) Py_RETURN_NONE;
  const at::Tensor *k = plain(a[0]), *v = plain(a[1]), *table = plain(a[3]);
  int64_t layer, length, stream;
  if (!k || !v || !table || !as_int(a[2], layer) || !as_int(a[4], length) || !as_int(a[5], stream)) Py_RETURN_NONE;
  const int code = dtype_code(k->scalar_type());
  if (k->dim() != 5 || code < 0 || v->scalar_type() != k->scalar_type() || v->sizes() != k->sizes() ||
      !k->is_contiguous() || !v->is_contiguous() || v->device() != k->device() || table->device() != k->device() ||
      table->scalar_type() != at::kInt || table->dim() != 1 || !table->is_contiguous())
    Py_RETURN_NONE;
  const auto s = k->sizes();
  const int64_t blocks = s[1], heads = s[2], block = s[3], dim = s[4];
  if (layer < 0 || layer >= s[0] || !fits(blocks) || !fits(heads) || !fits(block) || !fits(dim) || !fits(length) ||
      length > blocks * block || table->size(0) < blocks)
    Py_RETURN_NONE;
  const auto options = k->options().requires_grad(false);
  at::Tensor ko = at::empty({1, heads, length, dim}, options), vo = at::empty({1, heads, length, dim}, options);
  const int64_t tile = block * dim, offset = layer * blocks * heads * tile * k->element_size();
  const char* kp = static_cast<const char*>(k->data_ptr()) + offset;
  const char* vp = static_cast<const char*>(v->data_ptr()) + offset;
  const int32_t* tab = static_cast<const int32_t*>(table->data_ptr());
  void *kop = ko.data_ptr(), *vop = vo.data_ptr();
  int32_t rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_gather(kp, vp, heads * tile, tile, blocks, tab, length, kop, vop, length * dim, dim, heads, dim, block, code,
                reinterpret_cast<void*>(stream));
  Py_END_ALLOW_THREADS
  if (rc != MIE_OK) return PyLong_FromLong(rc);
  PyObject* pair = PyTuple_New(2);
  if (!pair) return nullptr;
  PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(std::move(ko)));
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(std::move(vo)));
  return pair;
  END_HANDLE_TH_ERRORS
}

// ---- a serving step's operators --------------------------------------------

// A vector of n values of this type on the device (any n if negative).
const at::Tensor* vec(PyObject* o, at::ScalarType type, c10::Device device, int64_t n) {
  const at::Tensor* t = plain(o);
  if (!t || t->dim() != 1 || t->scalar_type() != type || t->device() != device || !t->is_contiguous() ||
      (n >= 0 && t->size(0) != n))
    return nullptr;
  return t;
}

// The launch goes to the current device, and nothing is to be recorded.
bool usual(std::initializer_list<const at::Tensor*> tensors) {
  const at::Tensor& t = **tensors.begin();
  if (c10::impl::VirtualGuardImpl(t.device().type()).getDevice() != t.device()) return false;
  if (!c10::GradMode::is_enabled()) return true;
  for (const at::Tensor* x : tensors)
    if (x && x->requires_grad()) return false;
  return true;
}

bool as_double(PyObject* o, double& out) {
  if (PyFloat_CheckExact(o)) {
    out = PyFloat_AS_DOUBLE(o);
    return true;
  }
  int64_t i;
  if (!as_int(o, i)) return false;
  out = static_cast<double>(i);
  return true;
}

template <typename... T>
PyObject* pack(T&&... tensors) {
  PyObject* out = PyTuple_New(sizeof...(T));
  if (!out) return nullptr;
  Py_ssize_t i = 0;
  (PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(std::forward<T>(tensors))), ...);
  return out;
}

template <typename F>
int32_t released(F launch) {
  int32_t rc;
  Py_BEGIN_ALLOW_THREADS
  rc = launch();
  Py_END_ALLOW_THREADS
  return rc;
}

// n values of one allocation from the at-th on, as a tensor of their own: an
// at::empty costs 0.7 us, this 0.1.
at::Tensor piece(const at::Tensor& whole, int64_t at, int64_t n) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(), whole.dtype());
  impl->set_storage_offset(at);
  impl->set_sizes_contiguous({n});
  return at::Tensor(std::move(impl));
}

const int32_t* ints(const at::Tensor* t) { return t ? static_cast<const int32_t*>(t->data_ptr()) : nullptr; }
int32_t* ints_out(const at::Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }

// Block tables [B, n]: rows of int32, not overlapping.
const at::Tensor* table_rows(PyObject* o, c10::Device device) {
  const at::Tensor* t = plain(o);
  if (!t || t->dim() != 2 || t->scalar_type() != at::kInt || t->device() != device || t->size(0) < 1 ||
      t->size(1) < 1 || t->stride(1) != 1 || !fits(t->size(0)) || !fits(t->size(1)) ||
      (t->size(0) > 1 && t->stride(0) < t->size(1)))
    return nullptr;
  return t;
}

// reserve(free_ids, free_count, tables, context_lens, new_lens, block_size,
//         max_tokens, stream) -> six tensors, None or a status
PyObject* reserve(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) Py_RETURN_NONE;
  const at::Tensor* ids = plain(a[0]);
  int64_t block, tokens, stream;
  if (!ids || !as_int(a[5], block) || !as_int(a[6], tokens) || !as_int(a[7], stream)) Py_RETURN_NONE;
  const auto device = ids->device();
  const at::Tensor* tables = table_rows(a[2], device);
  if (!tables || !vec(a[0], at::kInt, device, -1)) Py_RETURN_NONE;
  const int64_t batch = tables->size(0);
  const at::Tensor *count = vec(a[1], at::kInt, device, 1), *lens = vec(a[3], at::kInt, device, batch),
                   *news = vec(a[4], at::kInt, device, batch);
  if (!count || !lens || !news || !fits(ids->size(0)) || block < 1 || !fits(block) || !fits(tokens) || !usual({ids}))
    Py_RETURN_NONE;
  const auto word = ids->options().requires_grad(false);
  // One allocation of words, the positions first (16-byte aligned).
  at::Tensor slots = at::empty({tokens}, word.dtype(at::kLong)), words = at::empty({tokens + 2 * batch + 3}, word);
  at::Tensor positions = piece(words, 0, tokens), starts = piece(words, tokens, batch + 1),
             lens_out = piece(words, tokens + batch + 1, batch), count_out = piece(words, tokens + 2 * batch + 1, 1),
             status = piece(words, tokens + 2 * batch + 2, 1);
  const int32_t rc = released([&] {
    return g_reserve(ints(ids), ids->size(0), ints(count), static_cast<int32_t*>(tables->data_ptr()),
                     std::max(tables->stride(0), tables->size(1)), tables->size(1), ints(lens), ints(news), batch, block,
                     tokens, ints_out(starts), static_cast<int64_t*>(slots.data_ptr()), ints_out(positions),
                     ints_out(lens_out), ints_out(count_out), ints_out(status), reinterpret_cast<void*>(stream));
  });
  if (rc != MIE_OK) return PyLong_FromLong(rc);
  return pack(starts, slots, positions, lens_out, count_out, status);
  END_HANDLE_TH_ERRORS
}

// release(free_ids, free_count, tables, context_lens, finished, block_size,
//         stream) -> three tensors, None or a status
PyObject* release(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) Py_RETURN_NONE;
  const at::Tensor* ids = plain(a[0]);
  int64_t block, stream;
  if (!ids || !as_int(a[5], block) || !as_int(a[6], stream)) Py_RETURN_NONE;
  const auto device = ids->device();
  const at::Tensor* tables = table_rows(a[2], device);
  if (!tables || !vec(a[0], at::kInt, device, -1)) Py_RETURN_NONE;
  const int64_t batch = tables->size(0);
  const at::Tensor *count = vec(a[1], at::kInt, device, 1), *lens = vec(a[3], at::kInt, device, batch),
                   *finished = vec(a[4], at::kBool, device, batch);
  if (!count || !lens || !finished || !fits(ids->size(0)) || block < 1 || !fits(block) || !usual({ids})) Py_RETURN_NONE;
  const auto word = ids->options().requires_grad(false);
  at::Tensor words = at::empty({batch + 2}, word);
  at::Tensor lens_out = piece(words, 0, batch), count_out = piece(words, batch, 1), status = piece(words, batch + 1, 1);
  const int32_t rc = released([&] {
    return g_release(static_cast<int32_t*>(ids->data_ptr()), ids->size(0), ints(count), ints(tables),
                     std::max(tables->stride(0), tables->size(1)), tables->size(1), ints(lens),
                     static_cast<const uint8_t*>(finished->data_ptr()), batch, block, ints_out(lens_out),
                     ints_out(count_out), ints_out(status), reinterpret_cast<void*>(stream));
  });
  if (rc != MIE_OK) return PyLong_FromLong(rc);
  return pack(count_out, lens_out, status);
  END_HANDLE_TH_ERRORS
}

// rope_append(q, k, v, k_pool, v_pool, layer, slots, positions, frequencies,
//             interleaved, factor, stream) -> q rotated, None or a status
PyObject* rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 12) Py_RETURN_NONE;
  const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]), *kp = plain(a[3]), *vp = plain(a[4]);
  int64_t layer, stream;
  double factor;
  if (!q || !k || !v || !kp || !vp || !as_int(a[5], layer) || !PyBool_Check(a[9]) || !as_double(a[10], factor) ||
      !as_int(a[11], stream))
    Py_RETURN_NONE;
  const int code = dtype_code(kp->scalar_type());
  const auto device = kp->device();
  if (code < 0 || q->dim() != 3 || k->dim() != 3 || kp->dim() != 5 || vp->sizes() != kp->sizes() ||
      !kp->is_contiguous() || !vp->is_contiguous() || vp->device() != device || vp->scalar_type() != kp->scalar_type())
    Py_RETURN_NONE;
  const auto ps = kp->sizes();
  const int64_t tokens = q->size(0), heads = q->size(1), blocks = ps[1], kv_heads = ps[2], block = ps[3], dim = ps[4];
  for (const at::Tensor* t : {q, k, v})
    if (t->scalar_type() != kp->scalar_type() || t->device() != device) Py_RETURN_NONE;
  if (q->size(2) != dim || q->stride(2) != 1 || k->size(0) != tokens || k->size(1) != kv_heads || k->size(2) != dim ||
      k->stride(2) != 1 || v->sizes() != k->sizes() || v->strides() != k->strides() || layer < 0 || layer >= ps[0] ||
      !fits(tokens) || !fits(heads) || !fits(blocks) || !fits(block) || !fits(dim))
    Py_RETURN_NONE;
  const at::Tensor *slots = vec(a[6], at::kLong, device, tokens), *positions = vec(a[7], at::kInt, device, tokens),
                   *freq = vec(a[8], at::kDouble, device, -1);
  if (!slots || !positions || !freq || freq->size(0) > dim || !usual({q, k, v, freq})) Py_RETURN_NONE;
  at::Tensor out = at::empty({tokens, heads, dim}, q->options().requires_grad(false));
  const int64_t tile = block * dim, offset = layer * blocks * kv_heads * tile * kp->element_size();
  const int32_t rc = released([&] {
    return g_rope(q->data_ptr(), q->stride(0), q->stride(1), k->data_ptr(), v->data_ptr(), k->stride(0), k->stride(1),
                  static_cast<char*>(kp->data_ptr()) + offset, static_cast<char*>(vp->data_ptr()) + offset,
                  kv_heads * tile, tile, blocks, static_cast<const int64_t*>(slots->data_ptr()), ints(positions),
                  static_cast<const double*>(freq->data_ptr()), 2 * freq->size(0), a[9] == Py_True,
                  static_cast<float>(factor), tokens, heads, kv_heads, dim, block, out.data_ptr(), heads * dim, dim,
                  code, reinterpret_cast<void*>(stream));
  });
  if (rc != MIE_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// extend(q, k_pool, v_pool, layer, tables, starts, context_lens, max_new,
//        max_len, scale, softcap, slopes, window, prefix_lens, stream) -> out,
// None or a status.  scale a float or None; slopes, prefix_lens may be None.
PyObject* extend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 15) Py_RETURN_NONE;
  const at::Tensor *q = plain(a[0]), *kp = plain(a[1]), *vp = plain(a[2]);
  int64_t layer, max_new, max_len, window, stream;
  double scale = 0, softcap;
  if (!q || !kp || !vp || !as_int(a[3], layer) || !as_int(a[7], max_new) || !as_int(a[8], max_len) ||
      (a[9] != Py_None && !as_double(a[9], scale)) || !as_double(a[10], softcap) || !as_int(a[12], window) ||
      !as_int(a[14], stream))
    Py_RETURN_NONE;
  const int code = dtype_code(q->scalar_type());
  const auto device = q->device();
  if (code < 0 || q->dim() != 3 || kp->dim() != 5 || vp->sizes() != kp->sizes() || !kp->is_contiguous() ||
      !vp->is_contiguous() || kp->device() != device || vp->device() != device ||
      kp->scalar_type() != q->scalar_type() || vp->scalar_type() != q->scalar_type())
    Py_RETURN_NONE;
  const auto ps = kp->sizes();
  const int64_t tokens = q->size(0), heads = q->size(1), blocks = ps[1], kv_heads = ps[2], block = ps[3], dim = ps[4];
  const int64_t align = 16 / q->element_size();
  const at::Tensor* tables = table_rows(a[4], device);
  if (!tables || tokens < 1 || q->size(2) != dim || q->stride(2) != 1 || q->stride(0) % align ||
      q->stride(1) % align || reinterpret_cast<uintptr_t>(q->data_ptr()) % 16 || layer < 0 || layer >= ps[0] ||
      kv_heads < 1 || heads < 1 || heads % kv_heads || !fits(tokens) || !fits(heads) || !fits(blocks) || !fits(block) ||
      !fits(dim) || !fits(max_new) || !fits(max_len) || !fits(window) || !(softcap >= 0 && std::isfinite(softcap)))
    Py_RETURN_NONE;
  const int64_t batch = tables->size(0);
  const at::Tensor *starts = vec(a[5], at::kInt, device, batch + 1), *lens = vec(a[6], at::kInt, device, batch),
                   *slopes = nullptr, *prefix = nullptr;
  if (!starts || !lens || (a[11] != Py_None && !(slopes = vec(a[11], at::kFloat, device, heads))) ||
      (a[13] != Py_None && !(prefix = vec(a[13], at::kInt, device, batch))) || !usual({q, kp, vp, slopes}))
    Py_RETURN_NONE;
  if (a[9] == Py_None) scale = 1.0 / std::sqrt(static_cast<double>(dim));
  const int64_t bytes = g_extend_workspace(tokens, batch, max_new, max_len, window, heads, kv_heads, dim, code);
  if (bytes < 0) Py_RETURN_NONE;  // refused: the other path says why
  at::Tensor out = at::empty({tokens, heads, dim}, q->options().requires_grad(false)), ws;
  if (bytes > 0) ws = at::empty({bytes}, q->options().dtype(at::kByte).requires_grad(false));
  const int64_t tile = block * dim, offset = layer * blocks * kv_heads * tile * kp->element_size();
  const int32_t rc = released([&] {
    return g_extend(q->data_ptr(), q->stride(0), q->stride(1), static_cast<const char*>(kp->data_ptr()) + offset,
                    static_cast<const char*>(vp->data_ptr()) + offset, kv_heads * tile, tile, blocks, ints(tables),
                    std::max(tables->stride(0), tables->size(1)), tables->size(1), ints(starts), ints(lens), tokens,
                    batch, max_new, max_len, heads, kv_heads, dim, block, static_cast<float>(scale),
                    static_cast<float>(softcap), slopes ? static_cast<const float*>(slopes->data_ptr()) : nullptr,
                    window, ints(prefix), out.data_ptr(), heads * dim, dim, bytes > 0 ? ws.data_ptr() : nullptr, bytes,
                    code, reinterpret_cast<void*>(stream));
  });
  if (rc != MIE_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// logprobs(logits, tokens, top, stream) -> (logprobs, entropy, top_logprobs,
// top_tokens), None or a status
PyObject* logprobs(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4) Py_RETURN_NONE;
  const at::Tensor* x = plain(a[0]);
  int64_t top, stream;
  if (!x || !as_int(a[2], top) || !as_int(a[3], stream)) Py_RETURN_NONE;
  const int code = dtype_code(x->scalar_type());
  if (code < 0 || x->dim() != 2) Py_RETURN_NONE;
  const int64_t rows = x->size(0), vocab = x->size(1);
  const at::Tensor* tokens = vec(a[1], at::kLong, x->device(), rows);
  if (!tokens || vocab < 1 || x->stride(1) != 1 || (rows > 1 && x->stride(0) < vocab) || !fits(rows) || !fits(vocab) ||
      top < 0 || top > vocab || !fits(top) || !usual({x}))
    Py_RETURN_NONE;
  const int64_t bytes = g_logprobs_workspace(rows, vocab, top);
  const auto real = x->options().dtype(at::kFloat).requires_grad(false);
  at::Tensor given = at::empty({rows}, real), entropy = at::empty({rows}, real), best = at::empty({rows, top}, real),
             ids = at::empty({rows, top}, real.dtype(at::kLong)), ws;
  if (bytes > 0) ws = at::empty({bytes}, real.dtype(at::kByte));
  const int32_t rc = released([&] {
    return g_logprobs(x->data_ptr(), std::max(x->stride(0), vocab), rows, vocab,
                      static_cast<const int64_t*>(tokens->data_ptr()), top, static_cast<float*>(given.data_ptr()),
                      static_cast<float*>(entropy.data_ptr()), static_cast<float*>(best.data_ptr()),
                      static_cast<int64_t*>(ids.data_ptr()), bytes > 0 ? ws.data_ptr() : nullptr, bytes, code,
                      reinterpret_cast<void*>(stream));
  });
  if (rc != MIE_OK) return PyLong_FromLong(rc);
  return pack(given, entropy, best, ids);
  END_HANDLE_TH_ERRORS
}

// bind(decode, decode_append, plan, plan_known, gather, reserve, release,
// rope_append, extend_workspace, extend, logprobs_workspace, logprobs): the
// entry points' addresses.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr int kEntries = 12;
  void* p[kEntries];
  if (n != kEntries) {
    PyErr_SetString(PyExc_TypeError, "bind takes twelve addresses");
    return nullptr;
  }
  for (int i = 0; i < kEntries; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: null address");
      return nullptr;
    }
  }
  g_decode = reinterpret_cast<decltype(g_decode)>(p[0]);
  g_decode_append = reinterpret_cast<decltype(g_decode_append)>(p[1]);
  g_plan = reinterpret_cast<decltype(g_plan)>(p[2]);
  g_plan_known = reinterpret_cast<decltype(g_plan_known)>(p[3]);
  g_gather = reinterpret_cast<decltype(g_gather)>(p[4]);
  g_reserve = reinterpret_cast<decltype(g_reserve)>(p[5]);
  g_release = reinterpret_cast<decltype(g_release)>(p[6]);
  g_rope = reinterpret_cast<decltype(g_rope)>(p[7]);
  g_extend_workspace = reinterpret_cast<decltype(g_extend_workspace)>(p[8]);
  g_extend = reinterpret_cast<decltype(g_extend)>(p[9]);
  g_logprobs_workspace = reinterpret_cast<decltype(g_logprobs_workspace)>(p[10]);
  g_logprobs = reinterpret_cast<decltype(g_logprobs)>(p[11]);
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(decode)), METH_FASTCALL, nullptr},
    {"gather", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(gather)), METH_FASTCALL, nullptr},
    {"reserve", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(reserve)), METH_FASTCALL, nullptr},
    {"release", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(release)), METH_FASTCALL, nullptr},
    {"rope_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(rope_append)), METH_FASTCALL, nullptr},
    {"extend", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(extend)), METH_FASTCALL, nullptr},
    {"logprobs", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(logprobs)), METH_FASTCALL, nullptr},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_host_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// abi_version: the header's version these calls were compiled for; bind() is
// for a library of the same one.
PyMODINIT_FUNC PyInit__host_calls() {
  PyObject* m = PyModule_Create(&g_module);
  if (m && PyModule_AddIntConstant(m, "abi_version", MIE_ABI_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
