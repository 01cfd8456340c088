// The calls over a 4-bit pool, those over an 8-bit pool, rotary positions and
// the copies of pages from Python without the interpreter's share: a CPython
// module over the tensors themselves. A call checks what its wrapper in
// ops_fp4.py, ops_fp8.py or ops.py checks, then calls the C entry point on the current stream.
// Whatever it finds different from the plain case (a check that fails, another
// current device, a tensor subclass, an exception) it leaves to the wrapper:
// it returns kNotTaken and has launched nothing, and the wrapper checks again
// and raises, or makes the call itself. So errors have one source.
//
// Host time of a call, this way and through the wrapper's checks and ctypes:
// decode 2.9 and 8.3 us, append 2.9 and 7.6, a read with its outputs' allocation
// 4.9 and 11.6; the launch is 2 to 3 of each. Rotary positions with their
// outputs' allocation 5 and 26 (Python's checks of eleven tensors), a copy of
// pages and the tables behind it 6 and 24.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <climits>

#include "nvk_paged_kv.h"

namespace {

constexpr long kNotTaken = 1;  // the entry points' codes are 0 or negative
constexpr int64_t kHeadDim = 128;

decltype(&nvk_fp4_append) entry_append = nullptr;
decltype(&nvk_fp4_read) entry_read = nullptr;
decltype(&nvk_fp4_qk_norm_rope_append) entry_norm = nullptr;
decltype(&nvk_fp4_paged_decode_reporting) entry_decode = nullptr;
decltype(&nvk_fp4_paged_prefill) entry_prefill = nullptr;
decltype(&nvk_fp8_append_workspace_size) entry_append8_workspace = nullptr;
decltype(&nvk_fp8_append) entry_append8 = nullptr;
decltype(&nvk_fp8_read) entry_read8 = nullptr;
decltype(&nvk_fp8_paged_decode) entry_decode8 = nullptr;
decltype(&nvk_fp8_paged_prefill) entry_prefill8 = nullptr;
decltype(&nvk_rotary) entry_rotary = nullptr;
decltype(&nvk_copy_blocks) entry_copy_blocks = nullptr;
decltype(&nvk_remap_blocks) entry_remap_blocks = nullptr;

struct Leave {};  // thrown where a call is left to the wrapper
void need(bool ok) {
  if (!ok) throw Leave{};
}

const at::Tensor& tensor(PyObject* o) {
  need(THPVariable_CheckExact(o));
  const at::Tensor& t = THPVariable_Unpack(o);
  need(t.defined() && t.layout() == at::kStrided);
  return t;
}
// A tensor on the device that the call runs on.
const at::Tensor& tensor_on(PyObject* o, c10::Device dev) {
  const at::Tensor& t = tensor(o);
  need(t.device() == dev);
  return t;
}
// The call's device: of its first tensor, a CUDA device and the current one.
c10::Device call_device(const at::Tensor& t) {
  const c10::Device dev = t.device();
  need(dev.is_cuda() && dev.index() == c10::cuda::current_device());
  return dev;
}
nvk_stream_t stream_on(c10::Device dev) {
  return reinterpret_cast<nvk_stream_t>(c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}
float number(PyObject* o) {
  if (PyFloat_CheckExact(o)) return static_cast<float>(PyFloat_AS_DOUBLE(o));
  need(PyLong_CheckExact(o));
  const double v = PyLong_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Leave{};
  }
  return static_cast<float>(v);
}
int to_int(int64_t v) {
  need(v >= 0 && v <= INT_MAX);
  return static_cast<int>(v);
}
int integer(PyObject* o) {
  need(PyLong_CheckExact(o));
  int overflow = 0;
  const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
  need(!overflow);
  return to_int(v);
}

struct Pool {
  void* data;
  int blocks, block_size, kv_heads;
};
Pool pool_of(const at::Tensor& t, int64_t unit_bytes = NVK_FP4_UNIT_BYTES) {
  static_assert(NVK_FP4_UNIT_TOKENS == NVK_FP8_UNIT_TOKENS, "a block size for both");
  need(t.scalar_type() == at::kByte && t.dim() == 4 && t.size(3) == unit_bytes && t.is_contiguous());
  return Pool{t.data_ptr(), to_int(t.size(0)), to_int(t.size(2) * NVK_FP4_UNIT_TOKENS), to_int(t.size(1))};
}
// The token stride of rows [tokens, heads, 128] whose heads and dims are packed.
int64_t rows(const at::Tensor& t) {
  need(t.dim() == 3 && t.size(2) == kHeadDim && t.stride(2) == 1 && t.stride(1) == kHeadDim);
  return t.stride(0);
}
int row_type(const at::Tensor& t) {
  need(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf);
  return t.scalar_type() == at::kHalf ? NVK_DTYPE_FP16 : NVK_DTYPE_BF16;
}
const at::Tensor& plain(const at::Tensor& t, at::ScalarType type, int64_t count) {
  need(t.scalar_type() == type && t.numel() == count && t.is_contiguous());
  return t;
}
int* error_ptr(PyObject* o, c10::Device dev) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor_on(o, dev);
  need(t.scalar_type() == at::kInt && t.numel() >= 1);
  return static_cast<int*>(t.data_ptr());
}
const int64_t* longs(const at::Tensor& t) { return static_cast<const int64_t*>(t.data_ptr()); }
const int32_t* ints(const at::Tensor& t) { return static_cast<const int32_t*>(t.data_ptr()); }

PyObject* pair_of(const at::Tensor& first, const at::Tensor& second) {
  PyObject *a = THPVariable_Wrap(first), *b = THPVariable_Wrap(second);
  PyObject* pair = a && b ? PyTuple_Pack(2, a, b) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  return pair;
}

template <typename Body>
PyObject* call(Py_ssize_t given, Py_ssize_t expected, Body&& body) {
  if (given != expected) {
    PyErr_Format(PyExc_TypeError, "%zd arguments, %zd expected", given, expected);
    return nullptr;
  }
  try {
    return body();
  } catch (...) {
    return PyLong_FromLong(kNotTaken);
  }
}

// append(kv_cache, key, value, slot_mapping, k_scale, v_scale, error_word)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 7, [&] {
    need(entry_append);
    const at::Tensor& cache = tensor(a[0]);
    const c10::Device dev = call_device(cache);
    const Pool p = pool_of(cache);
    const at::Tensor &key = tensor_on(a[1], dev), &value = tensor_on(a[2], dev);
    const int type = row_type(key);
    need(value.scalar_type() == key.scalar_type() && value.sizes() == key.sizes());
    const int64_t ks = rows(key), vs = rows(value), tokens = key.size(0);
    need(key.size(1) == p.kv_heads);
    const at::Tensor& slots = plain(tensor_on(a[3], dev), at::kLong, tokens);
    return PyLong_FromLong(entry_append(key.data_ptr(), value.data_ptr(), ks, vs, p.data, longs(slots), tokens,
                                        p.blocks, p.block_size, p.kv_heads, kHeadDim, type, number(a[4]),
                                        number(a[5]), error_ptr(a[6], dev), stream_on(dev)));
  });
}

// read(kv_cache, slot_mapping, k_scale, v_scale, half, error_word) -> (key, value), or a code
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 6, [&]() -> PyObject* {
    need(entry_read);
    const at::Tensor& cache = tensor(a[0]);
    const c10::Device dev = call_device(cache);
    const Pool p = pool_of(cache);
    const at::Tensor& slots = tensor_on(a[1], dev);
    const int64_t tokens = slots.numel();
    plain(slots, at::kLong, tokens);
    const float ks = number(a[2]), vs = number(a[3]);
    const bool half = a[4] == Py_True;
    int* err = error_ptr(a[5], dev);
    const auto options = at::TensorOptions().dtype(half ? at::kHalf : at::kBFloat16).device(dev);
    const at::Tensor key = at::empty({tokens, p.kv_heads, kHeadDim}, options), value = at::empty_like(key);
    const int rc = entry_read(key.data_ptr(), value.data_ptr(), p.data, longs(slots), tokens, p.blocks, p.block_size,
                              p.kv_heads, kHeadDim, half ? NVK_DTYPE_FP16 : NVK_DTYPE_BF16, ks, vs, err,
                              stream_on(dev));
    return rc == NVK_OK ? pair_of(key, value) : PyLong_FromLong(rc);
  });
}

// norm_rope_append(query, key, value, q_weight, k_weight, eps, cos, sin, positions, kv_cache, slot_mapping, k_scale,
// v_scale, query_out, error_word) -> the rotated query, or a code
PyObject* norm_rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 15, [&]() -> PyObject* {
    need(entry_norm);
    const at::Tensor& query = tensor(a[0]);
    const c10::Device dev = call_device(query);
    const at::Tensor &key = tensor_on(a[1], dev), &value = tensor_on(a[2], dev);
    need(query.scalar_type() == at::kBFloat16 && key.scalar_type() == at::kBFloat16 &&
         value.scalar_type() == at::kBFloat16);
    const int64_t qs = rows(query), ks = rows(key), vs = rows(value), tokens = query.size(0);
    const Pool p = pool_of(tensor_on(a[9], dev));
    need(key.size(0) == tokens && key.size(1) == p.kv_heads && value.sizes() == key.sizes());
    const at::Tensor& wq = plain(tensor_on(a[3], dev), at::kBFloat16, kHeadDim);
    const at::Tensor& wk = plain(tensor_on(a[4], dev), at::kBFloat16, kHeadDim);
    const at::Tensor &cos = tensor_on(a[6], dev), &sin = tensor_on(a[7], dev);
    need(cos.dim() == 2 && cos.size(1) == kHeadDim && sin.sizes() == cos.sizes());
    plain(cos, at::kFloat, cos.numel());
    plain(sin, at::kFloat, cos.numel());
    const at::Tensor& pos = plain(tensor_on(a[8], dev), at::kLong, tokens);
    const at::Tensor& slots = plain(tensor_on(a[10], dev), at::kLong, tokens);
    const float eps = number(a[5]), kc = number(a[11]), vc = number(a[12]);
    int* err = error_ptr(a[14], dev);
    at::Tensor out;
    if (a[13] == Py_None) {
      out = at::empty(query.sizes(), query.options());
    } else {
      out = tensor_on(a[13], dev);
      need(out.sizes() == query.sizes());
      plain(out, at::kBFloat16, query.numel());
    }
    const int rc = entry_norm(query.data_ptr(), key.data_ptr(), value.data_ptr(), qs, ks, vs, wq.data_ptr(),
                              wk.data_ptr(), eps, static_cast<const float*>(cos.data_ptr()),
                              static_cast<const float*>(sin.data_ptr()), to_int(cos.size(0)), longs(pos),
                              out.data_ptr(), p.data, longs(slots), tokens, p.blocks, p.block_size,
                              to_int(query.size(1)), p.kv_heads, kHeadDim, kc, vc, err, stream_on(dev));
    if (rc != NVK_OK) return PyLong_FromLong(rc);
    if (a[13] == Py_None) return THPVariable_Wrap(out);
    Py_INCREF(a[13]);
    return a[13];
  });
}

struct Attention {
  const at::Tensor &out, &query;
  Pool pool;
  const int32_t *tables, *lens;
  int batch, table_stride, table_columns, heads;
};
Attention attention(PyObject* const* a, PyObject* lens_object, c10::Device dev, int64_t unit_bytes = NVK_FP4_UNIT_BYTES) {
  const at::Tensor &query = tensor(a[1]), &out = tensor_on(a[0], dev);
  need(query.scalar_type() == at::kBFloat16 && query.dim() == 3 && query.size(2) == kHeadDim &&
       query.is_contiguous() && out.sizes() == query.sizes());
  plain(out, at::kBFloat16, query.numel());
  const Pool p = pool_of(tensor_on(a[2], dev), unit_bytes);
  const at::Tensor& tables = tensor_on(a[3], dev);
  need(tables.scalar_type() == at::kInt && tables.dim() == 2 && tables.stride(1) == 1);
  const int64_t batch = tables.size(0);
  const at::Tensor& lens = plain(tensor_on(lens_object, dev), at::kInt, batch);
  return Attention{out, query, p, ints(tables), ints(lens), to_int(batch),
                   to_int(batch > 1 ? tables.stride(0) : tables.size(1)), to_int(tables.size(1)),
                   to_int(query.size(1))};
}

// decode(out, query, kv_cache, block_tables, context_lens, scale, workspace, num_ctas, k_scale, v_scale, error_word)
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 11, [&] {
    need(entry_decode);
    const c10::Device dev = call_device(tensor(a[1]));
    const Attention t = attention(a, a[4], dev);
    need(t.query.size(0) == t.batch);
    const at::Tensor& ws = tensor_on(a[6], dev);
    need(ws.is_contiguous());
    return PyLong_FromLong(entry_decode(t.out.data_ptr(), t.query.data_ptr(), t.pool.data, t.pool.blocks,
                                        t.pool.block_size, t.tables, t.table_stride, t.table_columns, t.lens, t.batch,
                                        t.heads, t.pool.kv_heads, kHeadDim, number(a[5]), number(a[8]), number(a[9]),
                                        integer(a[7]), ws.data_ptr(), ws.nbytes(), error_ptr(a[10], dev),
                                        stream_on(dev)));
  });
}

// prefill(out, query, kv_cache, block_tables, cu_seqlens_q, kv_lens, max_q_len, scale, k_scale, v_scale, error_word)
PyObject* prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 11, [&] {
    need(entry_prefill);
    const c10::Device dev = call_device(tensor(a[1]));
    const Attention t = attention(a, a[5], dev);
    const at::Tensor& cu = plain(tensor_on(a[4], dev), at::kInt, int64_t(t.batch) + 1);
    return PyLong_FromLong(entry_prefill(t.out.data_ptr(), t.query.data_ptr(), t.pool.data, t.pool.blocks,
                                         t.pool.block_size, t.tables, t.table_stride, t.table_columns, ints(cu),
                                         t.lens, t.batch, to_int(t.query.size(0)), integer(a[6]), t.heads,
                                         t.pool.kv_heads, kHeadDim, number(a[7]), number(a[8]), number(a[9]),
                                         error_ptr(a[10], dev), stream_on(dev)));
  });
}

// append8(kv_cache, key, value, slot_mapping, error_word)
PyObject* append8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 5, [&] {
    need(entry_append8);
    const at::Tensor& cache = tensor(a[0]);
    const c10::Device dev = call_device(cache);
    const Pool p = pool_of(cache, NVK_FP8_UNIT_BYTES);
    const at::Tensor &key = tensor_on(a[1], dev), &value = tensor_on(a[2], dev);
    const int type = row_type(key);
    need(value.scalar_type() == key.scalar_type() && value.sizes() == key.sizes());
    const int64_t ks = rows(key), vs = rows(value), tokens = key.size(0);
    need(key.size(1) == p.kv_heads);
    const at::Tensor& slots = plain(tensor_on(a[3], dev), at::kLong, tokens);
    int* err = error_ptr(a[4], dev);
    size_t bytes = 0;
    need(entry_append8_workspace(tokens, int64_t(p.blocks) * p.block_size, &bytes) == NVK_OK);
    at::Tensor ws;  // of this call alone: the allocator gives it out again in the stream's order
    if (bytes) ws = at::empty({static_cast<int64_t>(bytes)}, cache.options());
    return PyLong_FromLong(entry_append8(key.data_ptr(), value.data_ptr(), ks, vs, p.data, longs(slots), tokens,
                                         p.blocks, p.block_size, p.kv_heads, kHeadDim, type,
                                         bytes ? ws.data_ptr() : nullptr, bytes, err, stream_on(dev)));
  });
}

// read8(kv_cache, slot_mapping, half, error_word) -> (key, value), or a code
PyObject* read8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 4, [&]() -> PyObject* {
    need(entry_read8);
    const at::Tensor& cache = tensor(a[0]);
    const c10::Device dev = call_device(cache);
    const Pool p = pool_of(cache, NVK_FP8_UNIT_BYTES);
    const at::Tensor& slots = tensor_on(a[1], dev);
    const int64_t tokens = slots.numel();
    plain(slots, at::kLong, tokens);
    const bool half = a[2] == Py_True;
    int* err = error_ptr(a[3], dev);
    const auto options = at::TensorOptions().dtype(half ? at::kHalf : at::kBFloat16).device(dev);
    const at::Tensor key = at::empty({tokens, p.kv_heads, kHeadDim}, options), value = at::empty_like(key);
    const int rc = entry_read8(key.data_ptr(), value.data_ptr(), p.data, longs(slots), tokens, p.blocks, p.block_size,
                               p.kv_heads, kHeadDim, half ? NVK_DTYPE_FP16 : NVK_DTYPE_BF16, err, stream_on(dev));
    return rc == NVK_OK ? pair_of(key, value) : PyLong_FromLong(rc);
  });
}

// decode8(out, query, kv_cache, block_tables, context_lens, scale, workspace, num_ctas, error_word)
PyObject* decode8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 9, [&] {
    need(entry_decode8);
    const c10::Device dev = call_device(tensor(a[1]));
    const Attention t = attention(a, a[4], dev, NVK_FP8_UNIT_BYTES);
    need(t.query.size(0) == t.batch);
    const at::Tensor& ws = tensor_on(a[6], dev);
    need(ws.is_contiguous());
    return PyLong_FromLong(entry_decode8(t.out.data_ptr(), t.query.data_ptr(), t.pool.data, t.pool.blocks,
                                         t.pool.block_size, t.tables, t.table_stride, t.table_columns, t.lens, t.batch,
                                         t.heads, t.pool.kv_heads, kHeadDim, number(a[5]), integer(a[7]),
                                         ws.data_ptr(), ws.nbytes(), error_ptr(a[8], dev), stream_on(dev)));
  });
}

// prefill8(out, query, kv_cache, block_tables, cu_seqlens_q, kv_lens, max_q_len, scale, error_word)
PyObject* prefill8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 9, [&] {
    need(entry_prefill8);
    const c10::Device dev = call_device(tensor(a[1]));
    const Attention t = attention(a, a[5], dev, NVK_FP8_UNIT_BYTES);
    const at::Tensor& cu = plain(tensor_on(a[4], dev), at::kInt, int64_t(t.batch) + 1);
    return PyLong_FromLong(entry_prefill8(t.out.data_ptr(), t.query.data_ptr(), t.pool.data, t.pool.blocks,
                                          t.pool.block_size, t.tables, t.table_stride, t.table_columns, ints(cu),
                                          t.lens, t.batch, to_int(t.query.size(0)), integer(a[6]), t.heads,
                                          t.pool.kv_heads, kHeadDim, number(a[7]), error_ptr(a[8], dev),
                                          stream_on(dev)));
  });
}

// rotary(query, key, inv_freq, positions, interleaved, attention_scale, q_weight, k_weight, eps, query_out, key_out)
// -> (query_out, key_out), or a code
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 11, [&]() -> PyObject* {
    need(entry_rotary);
    const at::Tensor& query = tensor(a[0]);
    const c10::Device dev = call_device(query);
    const at::Tensor& key = tensor_on(a[1], dev);
    const int type = row_type(query);
    need(key.scalar_type() == query.scalar_type() && query.dim() == 3 && key.dim() == 3);
    const int64_t tokens = query.size(0), dim = query.size(2);
    need(key.size(0) == tokens && key.size(2) == dim);
    auto stride = [&](const at::Tensor& t) {  // between tokens, of rows whose heads and dims are packed
      need(t.stride(2) == 1 && t.stride(1) == dim);
      return t.stride(0);
    };
    const at::Tensor& inv = tensor_on(a[2], dev);
    need(inv.dim() == 1 && inv.numel() > 0 && 2 * inv.numel() <= dim);
    plain(inv, at::kDouble, inv.numel());
    const at::Tensor& pos = plain(tensor_on(a[3], dev), at::kLong, tokens);
    need(PyBool_Check(a[4]) && (a[6] == Py_None) == (a[7] == Py_None));
    const void *wq = nullptr, *wk = nullptr;
    if (a[6] != Py_None) {
      wq = plain(tensor_on(a[6], dev), query.scalar_type(), dim).data_ptr();
      wk = plain(tensor_on(a[7], dev), query.scalar_type(), dim).data_ptr();
    }
    auto out_of = [&](PyObject* o, const at::Tensor& like) {
      if (o == Py_None) return at::empty(like.sizes(), like.options());
      const at::Tensor& t = tensor_on(o, dev);
      need(t.sizes() == like.sizes() && t.scalar_type() == like.scalar_type());
      return t;
    };
    const at::Tensor q_out = out_of(a[9], query), k_out = out_of(a[10], key);
    const int rc = entry_rotary(q_out.data_ptr(), k_out.data_ptr(), query.data_ptr(), key.data_ptr(), stride(q_out),
                                stride(k_out), stride(query), stride(key), wq, wk, number(a[8]),
                                static_cast<const double*>(inv.data_ptr()), longs(pos), number(a[5]), tokens,
                                to_int(query.size(1)), to_int(key.size(1)), to_int(dim), to_int(2 * inv.numel()),
                                a[4] == Py_True, type, stream_on(dev));
    return rc == NVK_OK ? pair_of(q_out, k_out) : PyLong_FromLong(rc);
  });
}

// copy_blocks(pool, second pool or None, pairs, error_word)
PyObject* copy_blocks(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 4, [&] {
    need(entry_copy_blocks);
    const at::Tensor& pool = tensor(a[0]);
    const c10::Device dev = call_device(pool);
    need(pool.dim() >= 3 && pool.is_contiguous() && pool.numel() > 0);
    void* second = nullptr;
    if (a[1] != Py_None) {
      const at::Tensor& t = tensor_on(a[1], dev);
      need(t.sizes() == pool.sizes() && t.scalar_type() == pool.scalar_type() && t.is_contiguous());
      second = t.data_ptr();
    }
    const at::Tensor& pairs = tensor_on(a[2], dev);
    need(pairs.dim() == 2 && pairs.size(1) == 2 && pairs.size(0) > 0);
    plain(pairs, at::kInt, pairs.numel());
    return PyLong_FromLong(entry_copy_blocks(pool.data_ptr(), second, to_int(pool.size(0)), to_int(pool.size(1)),
                                             static_cast<int64_t>(pool.nbytes()) / (pool.size(0) * pool.size(1)),
                                             ints(pairs), to_int(pairs.size(0)), error_ptr(a[3], dev),
                                             stream_on(dev)));
  });
}

// remap_blocks(block_tables, block_map, error_word)
PyObject* remap_blocks(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(n, 3, [&] {
    need(entry_remap_blocks);
    const at::Tensor& tables = tensor(a[0]);
    const c10::Device dev = call_device(tables);
    need(tables.scalar_type() == at::kInt && tables.dim() == 2 && tables.stride(1) == 1);
    const at::Tensor& map = tensor_on(a[1], dev);
    need(map.dim() == 1 && map.numel() > 0);
    plain(map, at::kInt, map.numel());
    return PyLong_FromLong(entry_remap_blocks(static_cast<int32_t*>(tables.data_ptr()),
                                              tables.size(0) > 1 ? tables.stride(0) : tables.size(1), tables.size(0),
                                              to_int(tables.size(1)), ints(map), to_int(map.numel()),
                                              error_ptr(a[2], dev), stream_on(dev)));
  });
}

// bind_more(append8's workspace size, append8, read8, decode8, prefill8, rotary, copy_blocks, remap_blocks): as bind
PyObject* bind_more(PyObject*, PyObject* args) {
  unsigned long long e[8];
  if (!PyArg_ParseTuple(args, "KKKKKKKK", &e[0], &e[1], &e[2], &e[3], &e[4], &e[5], &e[6], &e[7])) return nullptr;
  entry_append8_workspace = reinterpret_cast<decltype(entry_append8_workspace)>(e[0]);
  entry_append8 = reinterpret_cast<decltype(entry_append8)>(e[1]);
  entry_read8 = reinterpret_cast<decltype(entry_read8)>(e[2]);
  entry_decode8 = reinterpret_cast<decltype(entry_decode8)>(e[3]);
  entry_prefill8 = reinterpret_cast<decltype(entry_prefill8)>(e[4]);
  entry_rotary = reinterpret_cast<decltype(entry_rotary)>(e[5]);
  entry_copy_blocks = reinterpret_cast<decltype(entry_copy_blocks)>(e[6]);
  entry_remap_blocks = reinterpret_cast<decltype(entry_remap_blocks)>(e[7]);
  Py_RETURN_NONE;
}

// bind(append, read, norm_rope_append, decode, prefill): the entry points' addresses in the loaded library
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long e[5];
  if (!PyArg_ParseTuple(args, "KKKKK", &e[0], &e[1], &e[2], &e[3], &e[4])) return nullptr;
  entry_append = reinterpret_cast<decltype(entry_append)>(e[0]);
  entry_read = reinterpret_cast<decltype(entry_read)>(e[1]);
  entry_norm = reinterpret_cast<decltype(entry_norm)>(e[2]);
  entry_decode = reinterpret_cast<decltype(entry_decode)>(e[3]);
  entry_prefill = reinterpret_cast<decltype(entry_prefill)>(e[4]);
  Py_RETURN_NONE;
}

template <typename F>
PyMethodDef fast(const char* name, F f) {
  return PyMethodDef{name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {fast("append", append),
                         fast("read", read),
                         fast("norm_rope_append", norm_rope_append),
                         fast("decode", decode),
                         fast("prefill", prefill),
                         fast("append8", append8),
                         fast("read8", read8),
                         fast("decode8", decode8),
                         fast("prefill8", prefill8),
                         fast("rotary", rotary),
                         fast("copy_blocks", copy_blocks),
                         fast("remap_blocks", remap_blocks),
                         {"bind_more", bind_more, METH_VARARGS, nullptr},
                         {"bind", bind, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fp4_calls", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__fp4_calls() {
  PyObject* m = PyModule_Create(&module);
  if (m) PyModule_AddIntConstant(m, "NOT_TAKEN", kNotTaken);
  if (m) PyModule_AddStringConstant(m, "TORCH_VERSION", TORCH_VERSION);  // that it was built for
  return m;
}
