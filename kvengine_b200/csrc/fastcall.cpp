// The short way from Python to the kernels of a sampling decode step.
//
// A step calls each of these ops once per layer or pass for a few microseconds of GPU
// work, and through ctypes a call's checks, conversions and output tensors take ten to
// twenty microseconds of Python. These functions make the same checks and the
// same C ABI call from C++. Each takes the op's arguments in order and returns
//   the op's result          where everything is as the op wants it,
//   the library's code (int) where the library refused the call,
//   None                     in every other case (another current device, a workspace that
//                            has to grow, anything the op refuses or handles otherwise):
//                            kvengine_b200/ops.py then takes the call from the start
//                            and raises what there is to raise.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/kvengine_b200.h"

namespace {

// The library's entry points, as bind() gets their addresses.
decltype(&kve_paged_tree_attn) f_tree_attn;
decltype(&kve_tree_attn_workspace_bytes) f_tree_attn_ws;
decltype(&kve_qkv_rope_append_fp8) f_rope_append;
decltype(&kve_kv_read_fp8) f_read;
decltype(&kve_sample_accept) f_sample;
decltype(&kve_sample_accept_workspace_bytes) f_sample_ws;
decltype(&kve_tree_sample_accept) f_tree_sample;
decltype(&kve_tree_sample_accept_workspace_bytes) f_tree_sample_ws;
decltype(&kve_kv_commit_path) f_commit;

// Thrown for "not here": the Python path takes the call.
struct Other {};

const at::Tensor& tensor(PyObject* o) {
  if (!THPVariable_Check(o)) throw Other();
  return THPVariable_Unpack(o);
}
int integer(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Other();
  }
  if (v < INT32_MIN || v > INT32_MAX) throw Other();
  return (int)v;
}
void need(bool ok) {
  if (!ok) throw Other();
}
int own_device(const at::Tensor& t) {
  need(t.is_cuda());
  const int dev = t.get_device();
  need(dev == c10::cuda::current_device());
  return dev;
}
void dense(const at::Tensor& t, at::ScalarType type, int dev) {
  need(t.scalar_type() == type && t.is_cuda() && t.get_device() == dev && t.is_contiguous());
}
int code_of(at::ScalarType t) {
  if (t == at::kFloat) return KVE_F32;
  need(t == at::kBFloat16);
  return KVE_BF16;
}
cudaStream_t stream(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }
int* status_of(PyObject* o, int dev) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o);
  dense(t, at::kInt, dev);
  need(t.numel() >= 1);
  return t.data_ptr<int>();
}
template <typename T>
T* at_ptr(const at::Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
// The workspace's address and size, where it is large enough.
void* space(PyObject* o, size_t bytes, int dev, size_t* size) {
  if (bytes == 0) return *size = 0, nullptr;
  need(o != Py_None);
  const at::Tensor& t = tensor(o);
  dense(t, at::kByte, dev);
  need((size_t)t.numel() >= bytes);
  *size = (size_t)t.numel();
  return t.data_ptr();
}
// The row stride of a [rows, cols] matrix with unit column stride.
int64_t row_stride(const at::Tensor& t, at::ScalarType type, int dev, int64_t rows, int64_t cols) {
  need(t.scalar_type() == type && t.is_cuda() && t.get_device() == dev && t.dim() == 2 && t.size(0) == rows && t.size(1) == cols);
  if (t.is_contiguous()) return cols;
  need((cols <= 1 || t.stride(1) == 1) && (rows <= 1 || t.stride(0) >= cols));
  return std::max(t.stride(0), cols);
}
void fp8_cache(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs, int dev) {
  dense(k, at::kFloat8_e4m3fn, dev);
  dense(v, at::kFloat8_e4m3fn, dev);
  dense(ks, at::kByte, dev);
  dense(vs, at::kByte, dev);
  const auto shape = k.sizes();
  need(v.sizes() == shape && ks.sizes() == shape.slice(0, shape.size() - 1) && vs.sizes() == ks.sizes());
}
at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const at::Tensor& like) {
  return at::empty(shape, like.options().dtype(type));
}
PyObject* result(int rc, PyObject* (*make)(const at::Tensor*), const at::Tensor* t) {
  return rc ? PyLong_FromLong(rc) : make(t);
}
template <int N>
PyObject* tuple(const at::Tensor* t) {
  PyObject* r = PyTuple_New(N);
  if (!r) return nullptr;
  for (int i = 0; i < N; ++i) {
    PyObject* x = THPVariable_Wrap(t[i]);
    if (!x) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i, x);
  }
  return r;
}
PyObject* single(const at::Tensor* t) { return THPVariable_Wrap(t[0]); }
PyObject* nothing(const at::Tensor*) { return PyLong_FromLong(0); }

// No C++ exception leaves: whatever is thrown, the Python path takes the call.
template <PyObject* (*F)(PyObject* const*)>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  (void)n;  // ops.py is the only caller, with every argument
  try {
    return F(args);
  } catch (...) {
  }
  Py_RETURN_NONE;
}

// q, pool_k, pool_v, block_tables, ctx_lens, q_lens, q_offsets, max_q_len, max_ctx, scale, tree_mask, k_scale, v_scale, out,
// workspace, status
PyObject* tree_attention(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]), &tables = tensor(a[3]), &ctx = tensor(a[4]),
                   &ql = tensor(a[5]), &qo = tensor(a[6]);
  const int dev = own_device(q);
  const auto type = q.scalar_type();
  const int code = code_of(type);
  dense(q, type, dev);
  for (const at::Tensor* t : {&tables, &ctx, &ql, &qo}) dense(*t, at::kInt, dev);
  need(q.dim() == 3 && k.dim() == 4 && tables.dim() == 2 && k.size(3) == q.size(2) && v.sizes() == k.sizes());
  const int64_t B = tables.size(0), nq = q.size(1), hd = q.size(2);
  need(ctx.numel() == B && ql.numel() == B && qo.numel() >= B);
  int kv_code = code;
  const uint8_t *ks = nullptr, *vs = nullptr;
  if (a[11] == Py_None && a[12] == Py_None) {
    dense(k, type, dev);
    dense(v, type, dev);
  } else {
    const at::Tensor &s = tensor(a[11]), &t = tensor(a[12]);
    need(type == at::kBFloat16);
    fp8_cache(k, v, s, t, dev);
    ks = at_ptr<uint8_t>(s);
    vs = at_ptr<uint8_t>(t);
    kv_code = KVE_FP8_E4M3;
  }
  const uint32_t* mask = nullptr;
  int words = 0;
  if (a[10] != Py_None) {
    const at::Tensor& t = tensor(a[10]);
    dense(t, at::kInt, dev);
    need(t.dim() == 2 && t.size(0) == q.size(0));
    mask = at_ptr<uint32_t>(t);
    words = (int)t.size(1);
  }
  const int max_q = integer(a[7]), max_ctx = integer(a[8]);
  const double scale = PyFloat_AsDouble(a[9]);
  if (scale == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Other();
  }
  size_t size;
  void* ws = space(a[14], f_tree_attn_ws((int)B, max_q, max_ctx, (int)nq, (int)k.size(2), (int)hd), dev, &size);
  int* status = status_of(a[15], dev);
  at::Tensor out = a[13] == Py_None ? at::empty(q.sizes(), q.options()) : tensor(a[13]);
  if (a[13] != Py_None) {
    dense(out, type, dev);
    need(out.sizes() == q.sizes());
  }
  const int rc = f_tree_attn(q.data_ptr(), code, k.data_ptr(), v.data_ptr(), kv_code, ks, vs, at_ptr<int32_t>(tables),
                             (int)tables.size(1), at_ptr<int32_t>(ctx), at_ptr<int32_t>(ql), at_ptr<int32_t>(qo), mask, words,
                             (int)B, (int)q.size(0), max_q, max_ctx, (int)nq, (int)k.size(2), (int)hd, (int)k.size(1), k.size(0),
                             (float)scale, out.data_ptr(), ws, size, status, stream(dev));
  return result(rc, single, &out);
}

// qkv, positions, slots, rope_cos, rope_sin, q_out, pool_k, pool_v, k_scale, v_scale, num_heads, num_kv_heads, head_dim, status
PyObject* qkv_rope_append_fp8(PyObject* const* a) {
  const at::Tensor &qkv = tensor(a[0]), &pos = tensor(a[1]), &slots = tensor(a[2]), &c = tensor(a[3]), &s = tensor(a[4]),
                   &q = tensor(a[5]), &k = tensor(a[6]), &v = tensor(a[7]), &ks = tensor(a[8]), &vs = tensor(a[9]);
  const int dev = own_device(qkv);
  const auto type = qkv.scalar_type();
  const int code = code_of(type), nq = integer(a[10]), nkv = integer(a[11]), hd = integer(a[12]);
  dense(qkv, type, dev);
  dense(q, type, dev);
  dense(pos, at::kInt, dev);
  dense(slots, at::kInt, dev);
  dense(c, at::kFloat, dev);
  dense(s, at::kFloat, dev);
  fp8_cache(k, v, ks, vs, dev);
  need(qkv.dim() == 2 && k.dim() == 4 && c.dim() == 2 && k.size(2) == nkv && k.size(3) == hd && c.size(1) * 2 == hd &&
       s.sizes() == c.sizes());
  const int64_t n = qkv.size(0);
  need(n <= INT32_MAX && qkv.size(1) == (int64_t)(nq + 2 * nkv) * hd && pos.numel() == n && slots.numel() == n &&
       q.numel() == n * nq * hd);
  const int rc = f_rope_append(qkv.data_ptr(), code, (int)n, nq, nkv, hd, at_ptr<int32_t>(pos), at_ptr<int32_t>(slots),
                               at_ptr<float>(c), at_ptr<float>(s), (int)c.size(0), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                               at_ptr<uint8_t>(ks), at_ptr<uint8_t>(vs), k.size(0) * k.size(1), status_of(a[13], dev),
                               stream(dev));
  return result(rc, nothing, nullptr);
}

// pool_k, pool_v, k_scale, v_scale, slot_ids, bf16 (1) or fp32 (0), status
PyObject* kv_read_fp8(PyObject* const* a) {
  const at::Tensor &k = tensor(a[0]), &v = tensor(a[1]), &ks = tensor(a[2]), &vs = tensor(a[3]), &slots = tensor(a[4]);
  const int dev = own_device(k);
  fp8_cache(k, v, ks, vs, dev);
  dense(slots, at::kLong, dev);
  need(k.dim() == 4 && slots.dim() == 1 && slots.size(0) <= INT32_MAX);
  const bool bf16 = integer(a[5]) != 0;
  int* status = status_of(a[6], dev);
  const auto type = bf16 ? at::kBFloat16 : at::kFloat;
  const at::Tensor out[2] = {fresh({slots.size(0), k.size(2), k.size(3)}, type, k), fresh({slots.size(0), k.size(2), k.size(3)}, type, k)};
  const int rc = f_read(k.data_ptr(), v.data_ptr(), at_ptr<uint8_t>(ks), at_ptr<uint8_t>(vs), at_ptr<int64_t>(slots),
                        (int)slots.size(0), (int)k.size(2), (int)k.size(3), k.size(0) * k.size(1), bf16 ? KVE_BF16 : KVE_F32,
                        out[0].data_ptr(), out[1].data_ptr(), status, stream(dev));
  return result(rc, tuple<2>, out);
}

// logits, drafts, uniforms, gumbel, temperature, draft_logits, workspace, status
PyObject* sample_accept(PyObject* const* a) {
  const at::Tensor &x = tensor(a[0]), &drafts = tensor(a[1]), &u = tensor(a[2]), &noise = tensor(a[3]), &t = tensor(a[4]);
  const int dev = own_device(x);
  const auto type = x.scalar_type();
  const int code = code_of(type);
  need(x.dim() == 3);
  const int64_t B = x.size(0), k = x.size(1) - 1, V = x.size(2);
  need(B <= INT32_MAX && V <= INT32_MAX);
  need(drafts.scalar_type() == at::kInt && drafts.is_cuda() && drafts.get_device() == dev && drafts.dim() == 2 &&
       drafts.size(0) == B && drafts.size(1) == k);
  int64_t stride = V;
  if (!x.is_contiguous()) {
    stride = x.stride(1);
    need((V <= 1 || x.stride(2) == 1) && (B <= 1 || x.stride(0) == (k + 1) * stride) && stride >= V);
  }
  const int64_t us = row_stride(u, at::kFloat, dev, B, k), gs = row_stride(noise, at::kFloat, dev, B, V);
  dense(t, at::kFloat, dev);
  need(t.numel() == B);
  const void* dl = nullptr;
  int64_t dlb = 0, dlj = 0;
  if (a[5] != Py_None) {
    const at::Tensor& d = tensor(a[5]);
    need(d.scalar_type() == type && d.is_cuda() && d.get_device() == dev && d.dim() == 3 && d.size(0) == B && d.size(1) == k &&
         d.size(2) == V && (V <= 1 || d.stride(2) == 1));
    dl = d.data_ptr();
    dlb = d.stride(0);
    dlj = d.stride(1);
  }
  size_t size;
  void* ws = space(a[6], f_sample_ws((int)B, (int)k, (int)V, dl != nullptr), dev, &size);
  int* status = status_of(a[7], dev);
  const at::Tensor out[3] = {fresh({B}, at::kInt, x), fresh({B, k + 1}, at::kInt, x), fresh({B, k + 1}, at::kFloat, x)};
  const int rc = f_sample(x.data_ptr(), code, stride, dl, dlb, dlj, at_ptr<int32_t>(drafts), drafts.stride(0), drafts.stride(1),
                          at_ptr<float>(u), us, at_ptr<float>(noise), gs, at_ptr<float>(t), (int)B, (int)k, (int)V,
                          at_ptr<int32_t>(out[0]), at_ptr<int32_t>(out[1]), at_ptr<float>(out[2]), ws, size, status, stream(dev));
  return result(rc, tuple<3>, out);
}

// logits, tokens, parents, q_lens, q_offsets, max_q_len, uniforms, gumbel, temperature, workspace, status
PyObject* tree_sample_accept(PyObject* const* a) {
  const at::Tensor &x = tensor(a[0]), &tokens = tensor(a[1]), &parents = tensor(a[2]), &ql = tensor(a[3]), &qo = tensor(a[4]),
                   &u = tensor(a[6]), &noise = tensor(a[7]), &t = tensor(a[8]);
  const int dev = own_device(x), max_q = integer(a[5]);
  const auto type = x.scalar_type();
  const int code = code_of(type);
  need(x.dim() == 2 && max_q >= 0);
  const int64_t N = x.size(0), V = x.size(1), B = ql.numel();
  need(N <= INT32_MAX && V <= INT32_MAX && B <= INT32_MAX);
  const int64_t stride = row_stride(x, type, dev, N, V), gs = row_stride(noise, at::kFloat, dev, B, V);
  for (const at::Tensor* i : {&tokens, &parents, &ql, &qo}) dense(*i, at::kInt, dev);
  dense(u, at::kFloat, dev);
  dense(t, at::kFloat, dev);
  need(tokens.numel() == N && parents.numel() == N && u.numel() == N && qo.numel() >= B && t.numel() == B);
  size_t size;
  void* ws = space(a[9], f_tree_sample_ws((int)N, (int)V), dev, &size);
  int* status = status_of(a[10], dev);
  const at::Tensor out[4] = {fresh({B}, at::kInt, x), fresh({B, max_q}, at::kInt, x), fresh({B, max_q}, at::kInt, x),
                             fresh({B, max_q}, at::kFloat, x)};
  const int rc = f_tree_sample(x.data_ptr(), code, stride, at_ptr<int32_t>(tokens), at_ptr<int32_t>(parents), at_ptr<int32_t>(ql),
                               at_ptr<int32_t>(qo), at_ptr<float>(u), at_ptr<float>(noise), gs, at_ptr<float>(t), (int)B, (int)N,
                               max_q, (int)V, at_ptr<int32_t>(out[0]), at_ptr<int32_t>(out[1]), at_ptr<int32_t>(out[2]),
                               at_ptr<float>(out[3]), ws, size, status, stream(dev));
  return result(rc, tuple<4>, out);
}

// pool_k, pool_v, block_tables, start_lens, path, n_accepted, k_scale, v_scale, status
PyObject* kv_commit_path(PyObject* const* a) {
  const at::Tensor &k = tensor(a[0]), &v = tensor(a[1]), &tables = tensor(a[2]), &start = tensor(a[3]), &path = tensor(a[4]),
                   &n = tensor(a[5]);
  const int dev = own_device(k);
  need(k.dim() == 5 && tables.dim() == 2 && path.dim() == 2);
  int code;
  uint8_t *ks = nullptr, *vs = nullptr;
  if (a[6] == Py_None && a[7] == Py_None) {
    code = code_of(k.scalar_type());
    dense(k, k.scalar_type(), dev);
    dense(v, k.scalar_type(), dev);
    need(v.sizes() == k.sizes());
  } else {
    const at::Tensor &s = tensor(a[6]), &t = tensor(a[7]);
    fp8_cache(k, v, s, t, dev);
    ks = at_ptr<uint8_t>(s);
    vs = at_ptr<uint8_t>(t);
    code = KVE_FP8_E4M3;
  }
  for (const at::Tensor* t : {&tables, &start, &path, &n}) dense(*t, at::kInt, dev);
  const int64_t B = tables.size(0);
  need(B <= INT32_MAX && path.size(0) == B && start.numel() == B && n.numel() == B);
  const int rc = f_commit(k.data_ptr(), v.data_ptr(), code, ks, vs, (int)k.size(0), k.size(1), (int)k.size(2), (int)k.size(3),
                          (int)k.size(4), at_ptr<int32_t>(tables), (int)tables.size(1), at_ptr<int32_t>(start),
                          at_ptr<int32_t>(path), (int)path.size(1), at_ptr<int32_t>(n), (int)B, status_of(a[8], dev), stream(dev));
  return result(rc, nothing, nullptr);
}

// bind(addresses...): the library's entry points, in the order of the variables above.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  void* at[9];
  if (n != 9) {
    PyErr_SetString(PyExc_TypeError, "bind takes nine addresses");
    return nullptr;
  }
  for (int i = 0; i < 9; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: a null address");
      return nullptr;
    }
  }
  f_tree_attn = (decltype(f_tree_attn))at[0];
  f_tree_attn_ws = (decltype(f_tree_attn_ws))at[1];
  f_rope_append = (decltype(f_rope_append))at[2];
  f_read = (decltype(f_read))at[3];
  f_sample = (decltype(f_sample))at[4];
  f_sample_ws = (decltype(f_sample_ws))at[5];
  f_tree_sample = (decltype(f_tree_sample))at[6];
  f_tree_sample_ws = (decltype(f_tree_sample_ws))at[7];
  f_commit = (decltype(f_commit))at[8];
  Py_RETURN_NONE;
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))guarded<name>, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {{"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},
                         METHOD(tree_attention),
                         METHOD(qkv_rope_append_fp8),
                         METHOD(kv_read_fp8),
                         METHOD(sample_accept),
                         METHOD(tree_sample_accept),
                         METHOD(kv_commit_path),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastcall(void) { return PyModule_Create(&module); }
