// Thin CPython binding of the calls whose time is the host's: argument checks, output and scratch
// allocation and the C-ABI call in one step.  A call whose arguments need more than that (copies of
// strided rows, host lists, an error message) returns None and takes the Python path of the same
// function, which does everything this does.
#include <Python.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/logkv_attention.h"
#include "../../include/logkv_beam.h"

namespace {

using TreeFn = int (*)(const logkv_layout_t*, const logkv_state_t*, const logkv_prefix_t*, const logkv_tree_args_t*,
                       void*, size_t, void*);
using BeamFn = int (*)(const logkv_beam_args_t*, void*, size_t, void*);
using BeamBytesFn = size_t (*)(int32_t, int32_t, int32_t, int32_t);

template <typename T>
T address(PyObject* o) {
  return reinterpret_cast<T>(PyLong_AsVoidPtr(o));
}

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

at::Tensor bytes(size_t n, const at::Tensor& like) {
  return at::empty({(int64_t)n}, like.options().dtype(at::kByte).requires_grad(false));
}

PyObject* failed(int rc) { return PyLong_FromLong(rc); }

bool wants_gradient(const at::Tensor& t) { return t.requires_grad() && at::GradMode::is_enabled(); }

// [B, heads, T, D] rows in dtype and on the device of `like`, 16-byte aligned, without a gradient to record.
bool rows_ok(const at::Tensor& t, const at::Tensor& like, int64_t heads, int64_t tokens) {
  if (t.dim() != 4 || t.size(0) != like.size(0) || t.size(1) != heads || t.size(2) != tokens ||
      t.size(3) != like.size(3) || t.scalar_type() != like.scalar_type() || t.device() != like.device() ||
      t.stride(3) != 1 || wants_gradient(t))
    return false;
  const uint64_t e = t.element_size();
  return ((reinterpret_cast<uint64_t>(t.const_data_ptr()) | (uint64_t)t.stride(0) * e | (uint64_t)t.stride(1) * e |
           (uint64_t)t.stride(2) * e) & 15) == 0;
}

// tree(fn, layout, state, prefix, status, keys, q, k, v, parents, recent_count, scale, qx, scratch bytes):
// the output, an error code, or None.  `keys`: the packed prefix's keys [B, G, capacity, D].
PyObject* tree(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 14) {
    PyErr_SetString(PyExc_TypeError, "tree takes 14 arguments");
    return nullptr;
  }
  const at::Tensor *keys = tensor(args[5]), *q = tensor(args[6]), *k = tensor(args[7]), *v = tensor(args[8]),
                   *p = tensor(args[9]);
  if (!keys || !q || !k || !v || !p || !keys->is_cuda() || q->dim() != 4) Py_RETURN_NONE;
  const int64_t B = keys->size(0), G = keys->size(1), D = keys->size(3), H = q->size(1), T = q->size(2);
  if (T < 1 || T > LOGKV_TREE_MAX_TOKENS || H < 1 || H % G || !rows_ok(*q, *keys, H, T) || !rows_ok(*k, *keys, G, T) ||
      !rows_ok(*v, *keys, G, T))
    Py_RETURN_NONE;
  const bool wide = p->scalar_type() == at::kLong;
  if ((!wide && p->scalar_type() != at::kInt) || p->device() != keys->device() || p->dim() < 1 || p->dim() > 2 ||
      p->size(-1) != T || p->stride(-1) != 1 || (p->dim() == 2 && p->size(0) != B) ||
      c10::cuda::current_device() != keys->get_device())
    Py_RETURN_NONE;
  logkv_tree_args_t x{};
  x.recent_count = (int32_t)PyLong_AsLong(args[10]);
  x.scale = (float)PyFloat_AsDouble(args[11]);
  x.qx = (float)PyFloat_AsDouble(args[12]);
  const size_t need = PyLong_AsSize_t(args[13]);
  if (PyErr_Occurred()) return nullptr;
  try {
    const at::Tensor out = at::empty({B, H, T, D}, keys->options().requires_grad(false)), ws = bytes(need, *keys);
    x.q = q->const_data_ptr();
    x.k_new = k->const_data_ptr();
    x.v_new = v->const_data_ptr();
    x.out = out.mutable_data_ptr();
    x.parents = p->const_data_ptr();
    for (int i = 0; i < 3; ++i) {
      x.q_strides[i] = q->stride(i);
      x.k_strides[i] = k->stride(i);
      x.v_strides[i] = v->stride(i);
    }
    x.parents_stride = p->dim() == 2 ? p->stride(0) : 0;
    x.parents_wide = wide;
    x.heads = (int32_t)H;
    x.tokens = (int32_t)T;
    x.status = address<int32_t*>(args[4]);
    const int rc = address<TreeFn>(args[0])(address<const logkv_layout_t*>(args[1]), address<const logkv_state_t*>(args[2]),
                                            address<const logkv_prefix_t*>(args[3]), &x, ws.mutable_data_ptr(), need,
                                            c10::cuda::getCurrentCUDAStream().stream());
    return rc ? failed(rc) : THPVariable_Wrap(out);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// beam(fn, bytes fn, logits, scores, k, keep_places): (scores, rows, tokens), an error code, or None.
PyObject* beam(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "beam takes 6 arguments");
    return nullptr;
  }
  const at::Tensor *x = tensor(args[2]), *s = tensor(args[3]);
  if (!x || !s || !PyLong_Check(args[4]) || x->dim() != 3 || !x->is_cuda() || x->stride(2) != 1) Py_RETURN_NONE;
  const long k = PyLong_AsLong(args[4]);
  const int keep = PyObject_IsTrue(args[5]);
  if (PyErr_Occurred()) return nullptr;
  const int64_t N = x->size(0), W = x->size(1), V = x->size(2);
  const bool f32 = x->scalar_type() == at::kFloat;
  if ((!f32 && x->scalar_type() != at::kBFloat16) || s->dim() != 2 || s->size(0) != N || s->size(1) != W ||
      s->scalar_type() != at::kFloat || s->device() != x->device() || !s->is_contiguous() || N < 1 || N * W > 65535 ||
      V >= (1LL << 31) || k < 1 || k > LOGKV_BEAM_MAX_K || (keep && k != W) || wants_gradient(*x) || wants_gradient(*s) ||
      c10::cuda::current_device() != x->get_device())
    Py_RETURN_NONE;
  const size_t need = address<BeamBytesFn>(args[1])((int32_t)N, (int32_t)W, (int32_t)V, (int32_t)k);
  if (!need) Py_RETURN_NONE;
  try {
    const auto opt = s->options().requires_grad(false);
    const at::Tensor scores = at::empty({N, k}, opt), rows = at::empty({N, k}, opt.dtype(at::kLong)),
                     tokens = at::empty({N, k}, opt.dtype(at::kLong)), ws = bytes(need, *s);
    logkv_beam_args_t a{};
    a.logits = x->const_data_ptr();
    a.scores = static_cast<const float*>(s->const_data_ptr());
    a.out_scores = static_cast<float*>(scores.mutable_data_ptr());
    a.out_rows = static_cast<int64_t*>(rows.mutable_data_ptr());
    a.out_tokens = static_cast<int64_t*>(tokens.mutable_data_ptr());
    a.n_stride = x->stride(0);
    a.w_stride = x->stride(1);
    a.dtype = f32 ? LOGKV_DTYPE_F32 : LOGKV_DTYPE_BF16;
    a.requests = (int32_t)N;
    a.width = (int32_t)W;
    a.vocab = (int32_t)V;
    a.k = (int32_t)k;
    a.keep_places = keep;
    const int rc = address<BeamFn>(args[0])(&a, ws.mutable_data_ptr(), need, c10::cuda::getCurrentCUDAStream().stream());
    if (rc) return failed(rc);
    return Py_BuildValue("(NNN)", THPVariable_Wrap(scores), THPVariable_Wrap(rows), THPVariable_Wrap(tokens));
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyMethodDef methods[] = {
    {"tree", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(tree)), METH_FASTCALL, nullptr},
    {"beam", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(beam)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
