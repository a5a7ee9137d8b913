// The host side of the 4-bit pool's, the block tables' and the shared prefixes'
// calls for the common case, as one Python call each: the arguments' checks, the outputs and the
// scratch, then the C entry.
//
// A step's smallest calls are bound by the host: of a single sequence's decode
// (14.1 us a call through ops.py and ctypes) the two kernels' launches are 4.6
// us, the rest is reading some forty tensor attributes from Python and
// converting arguments.  Every function here returns None for whatever it does
// not take - a wrong type, shape, stride, alignment or device, a subclass of
// Tensor, tensors on another device than the current one - and launches
// nothing then: ops.py goes on with its own checks, which hold the errors'
// wording and the copies that unusual strides need.  A C entry's failure comes
// back as its status, an int.  Allocations and launches may wait (for a lock, for
// memory, for room in the stream's launch queue), so they run without the
// interpreter's lock, as the calls through ctypes do.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <limits>

#include "pagedserve_b200.h"

namespace {

using at::ScalarType;
using at::Tensor;

constexpr int64_t kMaxHeadDim = 256;
constexpr int64_t kI32 = std::numeric_limits<int32_t>::max();

// An argument that is a plain CUDA tensor on device ``dev``, or null.
const Tensor* cuda_tensor(PyObject* o, int dev) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.get_device() == dev ? &t : nullptr;
}

// The same for an argument that may be None; false: neither.
bool optional_tensor(PyObject* o, int dev, const Tensor** t) {
  *t = o == Py_None ? nullptr : cuda_tensor(o, dev);
  return o == Py_None || *t != nullptr;
}

bool as_int(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  int over = 0;
  *v = PyLong_AsLongLongAndOverflow(o, &over);
  return over == 0 && *v >= -1 && *v <= kI32;
}

int dtype_code(ScalarType t) {
  switch (t) {
    case at::kFloat: return PSB_F32;
    case at::kHalf: return PSB_F16;
    case at::kBFloat16: return PSB_BF16;
    default: return -1;
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

struct Pool {
  const Tensor *codes, *params;
  int64_t layers, blocks, heads, block_size, dim;
  ScalarType dtype;
  int code;
};

bool read_pool(PyObject* codes, PyObject* params, int dev, Pool* p) {
  p->codes = cuda_tensor(codes, dev);
  p->params = cuda_tensor(params, dev);
  if (!p->codes || !p->params || p->codes->dim() != 6 || p->params->dim() != 6) return false;
  const auto c = p->codes->sizes(), q = p->params->sizes();
  p->dtype = p->params->scalar_type();
  p->code = dtype_code(p->dtype);
  if (p->codes->scalar_type() != at::kByte || p->code < 0 || c[3] != 2 || q[5] != 2) return false;
  for (int i = 0; i < 5; ++i)
    if (c[i] != q[i] || c[i] <= 0 || c[i] > kI32) return false;
  p->layers = c[0];
  p->blocks = c[1];
  p->heads = c[2];
  p->block_size = c[4];
  p->dim = 2 * c[5];
  return p->dim > 0 && p->dim <= kMaxHeadDim && p->codes->is_contiguous() && p->params->is_contiguous() &&
         aligned16(p->codes->data_ptr()) && aligned16(p->params->data_ptr());
}

bool read_layer(PyObject* o, const Pool& p, int64_t* layer) { return as_int(o, layer) && *layer >= 0 && *layer < p.layers; }

// Rows [T, heads, D] of the pool's type with unit stride along D.
bool rows_like(const Tensor* t, const Pool& p, int64_t heads) {
  return t && t->dim() == 3 && t->size(2) == p.dim && t->scalar_type() == p.dtype && t->stride(2) == 1 &&
         (heads < 0 || t->size(1) == heads) && t->size(0) <= kI32;
}

bool i32_vector(const Tensor* t, int64_t n) {
  return t && t->dim() == 1 && t->scalar_type() == at::kInt && (n < 0 || t->size(0) == n) && t->size(0) <= kI32 &&
         t->is_contiguous();
}

bool slots_like(const Tensor* t, int64_t n) {
  return t && t->dim() == 1 && t->scalar_type() == at::kLong && (n < 0 || t->size(0) == n) && t->size(0) <= kI32 &&
         t->is_contiguous();
}

bool flag_like(const Tensor* t) { return !t || (t->scalar_type() == at::kInt && t->numel() >= 1); }

int32_t* flag_ptr(const Tensor* t) { return t ? static_cast<int32_t*>(t->data_ptr()) : nullptr; }

Tensor new_tensor(at::IntArrayRef sizes, ScalarType dtype, int dev) {
  return Tensor(at::detail::empty_cuda(sizes, dtype, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(dev)), std::nullopt));
}

// Whether an output made like ``t`` is contiguous (empty_like keeps the order
// of a dense tensor's axes).
bool plain_order(const Tensor& t) { return t.is_contiguous() || !t.is_non_overlapping_and_dense(); }

psb_stream_t stream_of(int dev) {
  return reinterpret_cast<psb_stream_t>(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream());
}

// Lets other threads have the interpreter while it lives.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

PyObject* none() { Py_RETURN_NONE; }
PyObject* true_or(int status) { return status == PSB_OK ? Py_NewRef(Py_True) : PyLong_FromLong(status); }
PyObject* out_or(int status, PyObject* given, const Tensor& t) {
  if (status != PSB_OK) return PyLong_FromLong(status);
  return given != Py_None ? Py_NewRef(given) : THPVariable_Wrap(t);
}

// write(key, value, kv_codes, kv_params, slot_mapping, layer, error_flag) -> True
PyObject* write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) return none();
  const int dev = c10::cuda::current_device();
  Pool p;
  const Tensor* flag;
  int64_t layer;
  if (!read_pool(a[2], a[3], dev, &p) || !read_layer(a[5], p, &layer) || !optional_tensor(a[6], dev, &flag) ||
      !flag_like(flag))
    return none();
  const Tensor *k = cuda_tensor(a[0], dev), *v = cuda_tensor(a[1], dev), *slots = cuda_tensor(a[4], dev);
  if (!rows_like(k, p, p.heads) || !rows_like(v, p, p.heads) || k->size(0) != v->size(0) || !slots_like(slots, k->size(0)))
    return none();
  int status;
  {
    const Unlocked unlocked;
    status = psb_reshape_and_cache_int4(k->data_ptr(), k->stride(0), k->stride(1), v->data_ptr(), v->stride(0),
                                        v->stride(1), p.codes->data_ptr(), p.params->data_ptr(),
                                        static_cast<const int64_t*>(slots->data_ptr()), k->size(0), layer, p.layers,
                                        p.blocks, p.heads, p.block_size, p.dim, p.code, flag_ptr(flag), stream_of(dev));
  }
  return true_or(status);
  END_HANDLE_TH_ERRORS
}

// rope_write(query, key, value, cos, sin, kv_codes, kv_params, slot_mapping, layer, key_out, error_flag)
// -> (query_out, key_out), both new; key_out None: a new one, False: none
PyObject* rope_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11 || !(a[9] == Py_None || a[9] == Py_False)) return none();
  const int dev = c10::cuda::current_device();
  Pool p;
  const Tensor* flag;
  int64_t layer;
  if (!read_pool(a[5], a[6], dev, &p) || !read_layer(a[8], p, &layer) || !optional_tensor(a[10], dev, &flag) ||
      !flag_like(flag))
    return none();
  const Tensor *q = cuda_tensor(a[0], dev), *k = cuda_tensor(a[1], dev), *v = cuda_tensor(a[2], dev);
  const Tensor *cos = cuda_tensor(a[3], dev), *sin = cuda_tensor(a[4], dev), *slots = cuda_tensor(a[7], dev);
  if (!rows_like(q, p, -1) || !rows_like(k, p, p.heads) || !rows_like(v, p, p.heads) || !cos || !sin) return none();
  const int64_t t = q->size(0);
  if (k->size(0) != t || v->size(0) != t || !slots_like(slots, t) || q->size(1) <= 0 || q->size(1) > kI32) return none();
  for (const Tensor* c : {cos, sin})
    if (c->dim() != 2 || c->size(0) != t || c->size(1) != p.dim || c->scalar_type() != p.dtype || c->stride(1) != 1 ||
        c->stride(0) != cos->stride(0))
      return none();
  const bool keep = a[9] == Py_None;
  if (!plain_order(*q) || (keep && !plain_order(*k))) return none();
  Tensor qo, ko;
  int status;
  {
    const Unlocked unlocked;
    qo = new_tensor(q->sizes(), p.dtype, dev);
    if (keep) ko = new_tensor(k->sizes(), p.dtype, dev);
    status = psb_rope_reshape_and_cache_int4(
        q->data_ptr(), q->stride(0), q->stride(1), qo.data_ptr(), qo.stride(0), qo.stride(1), k->data_ptr(),
        k->stride(0), k->stride(1), keep ? ko.data_ptr() : nullptr, keep ? ko.stride(0) : 0, keep ? ko.stride(1) : 0,
        v->data_ptr(), v->stride(0), v->stride(1), cos->data_ptr(), sin->data_ptr(), cos->stride(0),
        p.codes->data_ptr(), p.params->data_ptr(), static_cast<const int64_t*>(slots->data_ptr()), t, q->size(1), layer,
        p.layers, p.blocks, p.heads, p.block_size, p.dim, p.code, flag_ptr(flag), stream_of(dev));
  }
  if (status != PSB_OK) return PyLong_FromLong(status);
  return Py_BuildValue("(NN)", THPVariable_Wrap(qo), keep ? THPVariable_Wrap(ko) : Py_NewRef(Py_None));
  END_HANDLE_TH_ERRORS
}

// gather(kv_codes, kv_params, slot_mapping, layer, error_flag) -> (key, value), new
PyObject* gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) return none();
  const int dev = c10::cuda::current_device();
  Pool p;
  const Tensor* flag;
  int64_t layer;
  if (!read_pool(a[0], a[1], dev, &p) || !read_layer(a[3], p, &layer) || !optional_tensor(a[4], dev, &flag) ||
      !flag_like(flag))
    return none();
  const Tensor* slots = cuda_tensor(a[2], dev);
  if (!slots_like(slots, -1)) return none();
  const int64_t t = slots->size(0);
  Tensor k, v;
  int status;
  {
    const Unlocked unlocked;
    k = new_tensor({t, p.heads, p.dim}, p.dtype, dev);
    v = new_tensor({t, p.heads, p.dim}, p.dtype, dev);
    status = psb_gather_cache_int4(p.codes->data_ptr(), p.params->data_ptr(),
                                   static_cast<const int64_t*>(slots->data_ptr()), k.data_ptr(), k.stride(0), k.stride(1),
                                   v.data_ptr(), v.stride(0), v.stride(1), t, layer, p.layers, p.blocks, p.heads,
                                   p.block_size, p.dim, p.code, flag_ptr(flag), stream_of(dev));
  }
  if (status != PSB_OK) return PyLong_FromLong(status);
  return Py_BuildValue("(NN)", THPVariable_Wrap(k), THPVariable_Wrap(v));
  END_HANDLE_TH_ERRORS
}

// What decode and prefill share: the tables, the scale, the scratch and the output.
struct Attention {
  const Tensor *tables, *ctx, *out, *ws, *flag;
  int64_t layer, max_context;
  double scale;
};

bool read_attention(PyObject* const* a, int dev, const Pool& p, int64_t batch, Attention* t) {
  // a: block_tables, context_lens, layer, scale, out, max_context, workspace, error_flag
  t->tables = cuda_tensor(a[0], dev);
  t->ctx = cuda_tensor(a[1], dev);
  if (!t->tables || t->tables->dim() != 2 || t->tables->scalar_type() != at::kInt || t->tables->size(0) != batch ||
      t->tables->stride(1) != 1 || !i32_vector(t->ctx, batch))
    return false;
  const int64_t width = t->tables->size(1) * p.block_size;
  if (width > kI32 || !read_layer(a[2], p, &t->layer)) return false;
  if (a[3] == Py_None) t->scale = 1.0 / std::sqrt(static_cast<double>(p.dim));
  else if (PyFloat_CheckExact(a[3])) t->scale = PyFloat_AS_DOUBLE(a[3]);
  else return false;
  if (a[5] == Py_None) t->max_context = width;
  else if (!as_int(a[5], &t->max_context) || t->max_context < 0 || t->max_context > width) return false;
  return optional_tensor(a[4], dev, &t->out) && optional_tensor(a[6], dev, &t->ws) &&
         optional_tensor(a[7], dev, &t->flag) && flag_like(t->flag) &&
         (!t->ws || (t->ws->is_contiguous() && aligned16(t->ws->data_ptr())));
}

// decode(query, kv_codes, kv_params, block_tables, context_lens, layer, scale, out, max_context, workspace,
//        error_flag) -> out
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11) return none();
  const int dev = c10::cuda::current_device();
  Pool p;
  const Tensor* q = cuda_tensor(a[0], dev);
  if (!q || !read_pool(a[1], a[2], dev, &p)) return none();
  // [B, Hq, D] or [B, Hq, 1, D]
  auto rows = [&](const Tensor& t) {
    const int64_t d = t.dim();
    return (d == 3 || (d == 4 && t.size(2) == 1)) && t.size(d - 1) == p.dim && t.stride(d - 1) == 1 &&
           t.scalar_type() == p.dtype;
  };
  if (!rows(*q)) return none();
  const int64_t batch = q->size(0), heads = q->size(1);
  Attention t;
  if (batch <= 0 || batch > kI32 || heads <= 0 || heads > kI32 || heads % p.heads ||
      !read_attention(a + 3, dev, p, batch, &t))
    return none();
  if (t.out ? !rows(*t.out) || t.out->size(0) != batch || t.out->size(1) != heads : !plain_order(*q)) return none();
  Tensor out;
  int status;
  {
    const Unlocked unlocked;
    out = t.out ? *t.out : new_tensor(q->sizes(), p.dtype, dev);
    const Tensor ws = t.ws ? *t.ws
                           : new_tensor({static_cast<int64_t>(psb_paged_decode_int4_workspace_size(
                                            batch, heads, p.heads, p.dim, p.block_size, t.max_context, p.code))},
                                        at::kByte, dev);
    status = psb_paged_decode_int4(q->data_ptr(), q->stride(0), q->stride(1), out.data_ptr(), out.stride(0), out.stride(1),
                                   p.codes->data_ptr(), p.params->data_ptr(),
                                   static_cast<const int32_t*>(t.tables->data_ptr()), t.tables->stride(0),
                                   static_cast<const int32_t*>(t.ctx->data_ptr()), batch, heads, t.layer, p.layers,
                                   p.blocks, p.heads, p.block_size, p.dim, p.code, t.max_context,
                                   static_cast<float>(t.scale), ws.data_ptr(), ws.nbytes(), flag_ptr(t.flag),
                                   stream_of(dev));
  }
  return out_or(status, a[7], out);
  END_HANDLE_TH_ERRORS
}

// prefill(q, kv_codes, kv_params, cu_seqlens, max_seqlen, block_tables, context_lens, layer, scale, out, max_context,
//         workspace, error_flag) -> out
PyObject* prefill(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13) return none();
  const int dev = c10::cuda::current_device();
  Pool p;
  const Tensor *q = cuda_tensor(a[0], dev), *cu = cuda_tensor(a[3], dev);
  int64_t most;
  if (!read_pool(a[1], a[2], dev, &p) || !rows_like(q, p, -1) || !i32_vector(cu, -1) || cu->size(0) < 1 ||
      !as_int(a[4], &most) || most < 0)
    return none();
  const int64_t total = q->size(0), heads = q->size(1), batch = cu->size(0) - 1;
  Attention t;
  if (heads <= 0 || heads > kI32 || heads % p.heads || !read_attention(a + 5, dev, p, batch, &t) || most > t.max_context)
    return none();
  if (t.out ? !rows_like(t.out, p, heads) || t.out->size(0) != total : !plain_order(*q)) return none();
  Tensor out;
  int status;
  {
    const Unlocked unlocked;
    out = t.out ? *t.out : new_tensor(q->sizes(), p.dtype, dev);
    const Tensor ws = t.ws ? *t.ws
                           : new_tensor({static_cast<int64_t>(psb_paged_prefill_int4_workspace_size(
                                            total, batch, heads, p.heads, p.dim, p.block_size, t.max_context, p.code))},
                                        at::kByte, dev);
    status = psb_paged_prefill_int4(q->data_ptr(), q->stride(0), q->stride(1), p.codes->data_ptr(), p.params->data_ptr(),
                                    static_cast<const int32_t*>(t.tables->data_ptr()), t.tables->stride(0),
                                    static_cast<const int32_t*>(t.ctx->data_ptr()), out.data_ptr(), out.stride(0),
                                    out.stride(1), static_cast<const int32_t*>(cu->data_ptr()), batch, total, most,
                                    t.max_context, heads, t.layer, p.layers, p.blocks, p.heads, p.block_size, p.dim,
                                    p.code, static_cast<float>(t.scale), ws.data_ptr(), ws.nbytes(), flag_ptr(t.flag),
                                    stream_of(dev));
  }
  return out_or(status, a[9], out);
  END_HANDLE_TH_ERRORS
}

// What extend and trim share: table_store, three plan rows, free_blocks, free_state.
struct Tables {
  const Tensor *store, *rows, *first, *second, *free, *state, *flag;
  int64_t batch;
};

bool read_tables(PyObject* const* a, PyObject* flag, int dev, Tables* t) {
  t->store = cuda_tensor(a[0], dev);
  t->rows = cuda_tensor(a[1], dev);
  t->first = cuda_tensor(a[2], dev);
  t->second = cuda_tensor(a[3], dev);
  t->free = cuda_tensor(a[4], dev);
  t->state = cuda_tensor(a[5], dev);
  if (!t->store || t->store->dim() != 2 || t->store->scalar_type() != at::kInt || t->store->stride(1) != 1 ||
      t->store->stride(0) < t->store->size(1) || t->store->size(0) > kI32 || t->store->size(1) > kI32)
    return false;
  if (!i32_vector(t->rows, -1)) return false;
  t->batch = t->rows->size(0);
  return t->batch > 0 && i32_vector(t->first, t->batch) && i32_vector(t->second, t->batch) && i32_vector(t->free, -1) &&
         t->free->size(0) > 0 && i32_vector(t->state, 4) && optional_tensor(flag, dev, &t->flag) && flag_like(t->flag);
}

int32_t* ints(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }

// extend(table_store, req_rows, starts, query_lens, free_blocks, free_state, total, block_size, out_width, error_flag)
// -> (cu_seqlens, context_lens, slot_mapping, positions, block_tables), new
PyObject* extend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10) return none();
  const int dev = c10::cuda::current_device();
  Tables t;
  int64_t total, block, width;
  if (!read_tables(a, a[9], dev, &t) || !as_int(a[6], &total) || total < 0 || !as_int(a[7], &block) || block <= 0)
    return none();
  if (a[8] == Py_None) width = t.store->size(1);
  else if (!as_int(a[8], &width)) return none();
  if (width <= 0) return none();
  Tensor cu, ctx, slots, pos, tables;
  int status;
  {
    const Unlocked unlocked;
    cu = new_tensor({t.batch + 1}, at::kInt, dev);
    ctx = new_tensor({t.batch}, at::kInt, dev);
    slots = new_tensor({total}, at::kLong, dev);
    pos = new_tensor({total}, at::kLong, dev);
    tables = new_tensor({t.batch, width}, at::kInt, dev);
    status = psb_extend_step(ints(*t.store), t.store->stride(0), t.store->size(0), t.store->size(1), ints(*t.rows),
                             ints(*t.first), ints(*t.second), t.batch, ints(*t.free), t.free->size(0), ints(*t.state),
                             total, block, ints(cu), ints(ctx), static_cast<int64_t*>(slots.data_ptr()),
                             static_cast<int64_t*>(pos.data_ptr()), ints(tables), width, flag_ptr(t.flag), stream_of(dev));
  }
  if (status != PSB_OK) return PyLong_FromLong(status);
  return Py_BuildValue("(NNNNN)", THPVariable_Wrap(cu), THPVariable_Wrap(ctx), THPVariable_Wrap(slots),
                       THPVariable_Wrap(pos), THPVariable_Wrap(tables));
  END_HANDLE_TH_ERRORS
}

// trim(table_store, req_rows, held_lens, keep_lens, free_blocks, free_state, block_size, error_flag) -> True
PyObject* trim(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) return none();
  const int dev = c10::cuda::current_device();
  Tables t;
  int64_t block;
  if (!read_tables(a, a[7], dev, &t) || !as_int(a[6], &block) || block <= 0) return none();
  int status;
  {
    const Unlocked unlocked;
    status = psb_trim_tables(ints(*t.store), t.store->stride(0), t.store->size(0), t.store->size(1), ints(*t.rows),
                             ints(*t.first), ints(*t.second), t.batch, ints(*t.free), t.free->size(0), ints(*t.state),
                             block, flag_ptr(t.flag), stream_of(dev));
  }
  return true_or(status);
  END_HANDLE_TH_ERRORS
}

// Holder counts: int32 [2, blocks of the ring].
bool shares_like(const Tensor* t, const Tables& of) {
  return t && t->dim() == 2 && t->scalar_type() == at::kInt && t->size(0) == 2 && t->size(1) == of.free->size(0) && t->is_contiguous();
}

// fork(table_store, parent_rows, child_rows, lens, free_blocks, free_state, shares, block_size, error_flag)
// -> (src, dst), new
PyObject* fork(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9) return none();
  const int dev = c10::cuda::current_device();
  Tables t;
  int64_t block;
  if (!read_tables(a, a[8], dev, &t) || !as_int(a[7], &block) || block <= 0) return none();
  const Tensor* shares = cuda_tensor(a[6], dev);
  if (!shares_like(shares, t)) return none();
  Tensor src, dst;
  int status;
  {
    const Unlocked unlocked;
    src = new_tensor({t.batch}, at::kInt, dev);
    dst = new_tensor({t.batch}, at::kInt, dev);
    status = psb_fork_tables(ints(*t.store), t.store->stride(0), t.store->size(0), t.store->size(1), ints(*t.rows),
                             ints(*t.first), ints(*t.second), t.batch, ints(*shares), ints(*t.free), t.free->size(0),
                             ints(*t.state), block, ints(src), ints(dst), flag_ptr(t.flag), stream_of(dev));
  }
  if (status != PSB_OK) return PyLong_FromLong(status);
  return Py_BuildValue("(NN)", THPVariable_Wrap(src), THPVariable_Wrap(dst));
  END_HANDLE_TH_ERRORS
}

// release(table_store, req_rows, held_lens, keep_lens, free_blocks, free_state, shares, block_size, error_flag) -> True
PyObject* release(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9) return none();
  const int dev = c10::cuda::current_device();
  Tables t;
  int64_t block;
  if (!read_tables(a, a[8], dev, &t) || !as_int(a[7], &block) || block <= 0) return none();
  const Tensor* shares = cuda_tensor(a[6], dev);
  if (!shares_like(shares, t)) return none();
  int status;
  {
    const Unlocked unlocked;
    status = psb_release_tables(ints(*t.store), t.store->stride(0), t.store->size(0), t.store->size(1), ints(*t.rows),
                                ints(*t.first), ints(*t.second), t.batch, ints(*shares), ints(*t.free), t.free->size(0),
                                ints(*t.state), block, flag_ptr(t.flag), stream_of(dev));
  }
  return true_or(status);
  END_HANDLE_TH_ERRORS
}

// copy(pools, src, dst, error_flag) -> True; pools: a tuple
PyObject* copy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4 || !PyTuple_CheckExact(a[0])) return none();
  const int dev = c10::cuda::current_device();
  const Py_ssize_t count = PyTuple_GET_SIZE(a[0]);
  const Tensor *src = cuda_tensor(a[1], dev), *dst = cuda_tensor(a[2], dev), *flag;
  if (count < 1 || count > 4 || !i32_vector(src, -1) || !i32_vector(dst, src->size(0)) || !optional_tensor(a[3], dev, &flag) ||
      !flag_like(flag))
    return none();
  void* pools[4];
  int64_t bytes[4], layers = 0, blocks = 0;
  for (Py_ssize_t i = 0; i < count; ++i) {
    const Tensor* const t = cuda_tensor(PyTuple_GET_ITEM(a[0], i), dev);
    if (!t || t->dim() < 3 || t->numel() == 0 || !t->is_contiguous() || t->size(0) > kI32 || t->size(1) > kI32) return none();
    if (i > 0 && (t->size(0) != layers || t->size(1) != blocks)) return none();
    layers = t->size(0);
    blocks = t->size(1);
    pools[i] = t->data_ptr();
    bytes[i] = static_cast<int64_t>(t->nbytes()) / (layers * blocks);
  }
  int status;
  {
    const Unlocked unlocked;
    status = psb_copy_blocks(pools, bytes, static_cast<int32_t>(count), ints(*src), ints(*dst), src->size(0), layers, blocks,
                             flag_ptr(flag), stream_of(dev));
  }
  return true_or(status);
  END_HANDLE_TH_ERRORS
}

// decode_shared(query, k_cache, v_cache, block_tables, context_lens, cu_groups, prefix_lens, layer, scale, out, max_context,
//               workspace, error_flag) -> out
PyObject* decode_shared(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 13) return none();
  const int dev = c10::cuda::current_device();
  const Tensor *q = cuda_tensor(a[0], dev), *k = cuda_tensor(a[1], dev), *v = cuda_tensor(a[2], dev);
  const Tensor *tables = cuda_tensor(a[3], dev), *ctx = cuda_tensor(a[4], dev), *cu = cuda_tensor(a[5], dev), *pre = cuda_tensor(a[6], dev);
  const Tensor *out, *ws, *flag;
  int64_t layer, most;
  if (!q || !k || !v || !tables || k->dim() != 5 || k->sizes() != v->sizes() || k->scalar_type() != v->scalar_type() ||
      !k->is_contiguous() || !v->is_contiguous() || k->numel() == 0 || !as_int(a[7], &layer) || layer < 0 || layer >= k->size(0))
    return none();
  const int64_t layers = k->size(0), blocks = k->size(1), hkv = k->size(2), block = k->size(3), dim = k->size(4);
  const ScalarType type = k->scalar_type();
  auto rows = [&](const Tensor& t) {
    const int64_t d = t.dim();
    return (d == 3 || (d == 4 && t.size(2) == 1)) && t.size(d - 1) == dim && t.stride(d - 1) == 1 && t.scalar_type() == type;
  };
  if ((type != at::kHalf && type != at::kBFloat16) || block > kI32 || layers * hkv > kI32 / blocks || !rows(*q)) return none();
  const int64_t batch = q->size(0), heads = q->size(1);
  if (batch <= 0 || batch > kI32 || heads <= 0 || heads > kI32 || heads % hkv || q->stride(0) <= 0 || q->stride(1) <= 0 ||
      q->stride(0) % 8 || q->stride(1) % 8 || !aligned16(q->data_ptr()) || !aligned16(k->data_ptr()) || !aligned16(v->data_ptr()))
    return none();
  if (tables->dim() != 2 || tables->scalar_type() != at::kInt || tables->size(0) != batch || tables->stride(1) != 1 || tables->stride(0) < 0 ||
      !i32_vector(ctx, batch) || !i32_vector(pre, -1) || !i32_vector(cu, pre->size(0) + 1) || tables->size(1) > kI32 / block)
    return none();
  const int64_t width = tables->size(1) * block;
  double scale;
  if (a[8] == Py_None) scale = 1.0 / std::sqrt(static_cast<double>(dim));
  else if (PyFloat_CheckExact(a[8])) scale = PyFloat_AS_DOUBLE(a[8]);
  else return none();
  if (!(scale > 0.0) || !std::isfinite(scale)) return none();
  if (a[10] == Py_None) most = width;
  else if (!as_int(a[10], &most) || most < 0 || most > width) return none();
  if (!optional_tensor(a[9], dev, &out) || !optional_tensor(a[11], dev, &ws) || !optional_tensor(a[12], dev, &flag) || !flag_like(flag) ||
      (ws && (!ws->is_contiguous() || !aligned16(ws->data_ptr()))))
    return none();
  if (out ? !rows(*out) || out->size(0) != batch || out->size(1) != heads : !plain_order(*q)) return none();
  const size_t need = psb_paged_decode_shared_workspace_size(batch, pre->size(0), heads, hkv, dim, block, most, dtype_code(type));
  if (need == 0) return none();
  Tensor o;
  int status;
  {
    const Unlocked unlocked;
    o = out ? *out : new_tensor(q->sizes(), type, dev);
    const Tensor w = ws ? *ws : new_tensor({static_cast<int64_t>(need)}, at::kByte, dev);
    status = psb_paged_decode_shared(q->data_ptr(), q->stride(0), q->stride(1), o.data_ptr(), o.stride(0), o.stride(1), k->data_ptr(),
                                     v->data_ptr(), ints(*tables), tables->stride(0), ints(*ctx), ints(*cu), ints(*pre), batch,
                                     pre->size(0), heads, layer, layers, blocks, hkv, block, dim, dtype_code(type), most,
                                     static_cast<float>(scale), w.data_ptr(), w.nbytes(), flag_ptr(flag), stream_of(dev));
  }
  return out_or(status, a[9], o);
  END_HANDLE_TH_ERRORS
}

// verify(logits, tokens, cu_seqlens, uniforms, temperature, draft_probs, error_flag) -> (new_tokens, counts), new
PyObject* verify(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) return none();
  const int dev = c10::cuda::current_device();
  const Tensor *x = cuda_tensor(a[0], dev), *tokens = cuda_tensor(a[1], dev), *cu = cuda_tensor(a[2], dev);
  const Tensor *u = cuda_tensor(a[3], dev), *heat = cuda_tensor(a[4], dev), *probs, *flag;
  if (!x || !u || !optional_tensor(a[5], dev, &probs) || !optional_tensor(a[6], dev, &flag) || !flag_like(flag) || x->dim() != 2)
    return none();
  const int64_t rows = x->size(0), vocab = x->size(1);
  auto matrix = [&](const Tensor& t) {
    return t.dim() == 2 && t.size(0) == rows && t.size(1) == vocab && t.stride(1) == 1 && t.stride(0) >= vocab && dtype_code(t.scalar_type()) >= 0;
  };
  if (rows <= 0 || rows > kI32 || vocab <= 0 || vocab > kI32 || !matrix(*x) || (probs && !matrix(*probs)) || !slots_like(tokens, rows) ||
      !i32_vector(cu, -1) || cu->size(0) < 2)
    return none();
  const int64_t batch = cu->size(0) - 1;
  if (u->scalar_type() != at::kFloat || u->dim() != 2 || u->size(0) != rows || u->size(1) != 2 || !u->is_contiguous() || !heat ||
      heat->scalar_type() != at::kFloat || heat->dim() != 1 || heat->size(0) != batch || !heat->is_contiguous())
    return none();
  Tensor fresh, counts;
  int status;
  {
    const Unlocked unlocked;
    fresh = new_tensor({rows}, at::kLong, dev);
    counts = new_tensor({batch}, at::kInt, dev);
    const Tensor ws = new_tensor({static_cast<int64_t>(psb_verify_tokens_workspace_size(batch))}, at::kByte, dev);
    status = psb_verify_tokens(x->data_ptr(), x->stride(0), rows, vocab, dtype_code(x->scalar_type()),
                               static_cast<const int64_t*>(tokens->data_ptr()), ints(*cu), batch, static_cast<const float*>(u->data_ptr()),
                               static_cast<const float*>(heat->data_ptr()), probs ? probs->data_ptr() : nullptr,
                               probs ? probs->stride(0) : 0, probs ? dtype_code(probs->scalar_type()) : 0,
                               static_cast<int64_t*>(fresh.data_ptr()), ints(counts), ws.data_ptr(), ws.nbytes(), flag_ptr(flag),
                               stream_of(dev));
  }
  if (status != PSB_OK) return PyLong_FromLong(status);
  return Py_BuildValue("(NN)", THPVariable_Wrap(fresh), THPVariable_Wrap(counts));
  END_HANDLE_TH_ERRORS
}

#define ENTRY(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(write), ENTRY(rope_write), ENTRY(gather), ENTRY(decode), ENTRY(prefill),
                         ENTRY(extend), ENTRY(trim), ENTRY(fork), ENTRY(release), ENTRY(copy),
                         ENTRY(decode_shared), ENTRY(verify), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() {
  PyObject* m = PyModule_Create(&module);
  // what it was compiled against (build.py's calls_target), for the loader to compare
  if (m != nullptr && PyModule_AddStringConstant(m, "built_for", PSB_BUILT_FOR) != 0) Py_CLEAR(m);
  return m;
}
