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

#include <cmath>

#include "../../include/logkv_attention.h"
#include "../../include/logkv_beam.h"
#include "../../include/logkv_logits.h"
#include "../../include/logkv_rotary.h"

namespace {

using TreeFn = int (*)(const logkv_layout_t*, const logkv_state_t*, const logkv_prefix_t*, const logkv_tree_args_t*,
                       void*, size_t, void*);
using BeamFn = int (*)(const logkv_beam_args_t*, void*, size_t, void*);
using BeamBytesFn = size_t (*)(int32_t, int32_t, int32_t, int32_t);
using SharedFn = int (*)(const logkv_layout_t*, const logkv_state_t*, const logkv_prefix_t*, const logkv_shared_args_t*,
                         void*, size_t, void*);
using SharedBytesFn = size_t (*)(const logkv_layout_t*, const logkv_shared_args_t*, int32_t);
using RotateFn = int (*)(const logkv_rope_t*, const logkv_rotate_args_t*, void*);
using LogitsFn = int (*)(const logkv_logits_args_t*, void*);

template <typename T>
T address(PyObject* o) {
  return reinterpret_cast<T>(PyLong_AsVoidPtr(o));
}

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

at::Tensor bytes(size_t n, const at::Tensor& like) {
  return at::empty({(int64_t)n}, like.options().dtype(at::kByte).requires_grad(false));
}

PyObject* failed(int rc) { return PyLong_FromLong(rc); }

// Whether the Python numbers read before fitted their C types; if not, the Python path says what is wrong with them.
bool in_range() {
  if (!PyErr_Occurred()) return true;
  PyErr_Clear();
  return false;
}

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

// shared(fn, bytes fn, layout, state, prefix, status, keys, q, k, v, recent_count, beams, window_from, causal tail
// or None, scale, qx): the output, an error code, or None.  `keys`: the packed prefix's keys [B, G, capacity, D].
PyObject* shared(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 16) {
    PyErr_SetString(PyExc_TypeError, "shared takes 16 arguments");
    return nullptr;
  }
  const at::Tensor *keys = tensor(args[6]), *q = tensor(args[7]), *k = tensor(args[8]), *v = tensor(args[9]);
  if (!keys || !q || !k || !v || !keys->is_cuda() || q->dim() != 4 || k->dim() != 4 || !PyLong_Check(args[10]) ||
      !PyLong_Check(args[11]) || !PyLong_Check(args[12]))
    Py_RETURN_NONE;
  const int64_t B = keys->size(0), G = keys->size(1), D = keys->size(3), H = q->size(1), T = q->size(2), Tk = k->size(2);
  if (T < 1 || Tk < T || Tk > INT32_MAX || H < 1 || H % G || !rows_ok(*q, *keys, H, T) || !rows_ok(*k, *keys, G, Tk) ||
      !rows_ok(*v, *keys, G, Tk) || c10::cuda::current_device() != keys->get_device())
    Py_RETURN_NONE;
  const long recent = PyLong_AsLong(args[10]), beams = PyLong_AsLong(args[11]), from = PyLong_AsLong(args[12]);
  long tail = T;
  if (args[13] != Py_None) {
    if (!PyLong_Check(args[13])) Py_RETURN_NONE;
    tail = PyLong_AsLong(args[13]);
  }
  if (!in_range()) Py_RETURN_NONE;
  logkv_shared_args_t x{};
  x.scale = (float)PyFloat_AsDouble(args[14]);
  x.qx = (float)PyFloat_AsDouble(args[15]);
  if (PyErr_Occurred()) return nullptr;
  if ((tail && (tail != T || T != Tk)) || beams < 1 || beams > B || B % beams || recent < 0 || recent > INT32_MAX ||
      from < 0 || from > recent)
    Py_RETURN_NONE;
  for (int i = 0; i < 3; ++i) {
    x.q_strides[i] = q->stride(i);
    x.k_strides[i] = k->stride(i);
    x.v_strides[i] = v->stride(i);
  }
  x.heads = (int32_t)H;
  x.beams = (int32_t)beams;
  x.q_tokens = (int32_t)T;
  x.tokens = (int32_t)Tk;
  x.recent_count = (int32_t)recent;
  x.window_from = (int32_t)from;
  x.causal = tail != 0;
  x.status = address<int32_t*>(args[5]);
  const auto* layout = address<const logkv_layout_t*>(args[2]);
  const auto* prefix = address<const logkv_prefix_t*>(args[4]);
  const size_t need = address<SharedBytesFn>(args[1])(layout, &x, prefix->capacity);
  if (!need) Py_RETURN_NONE;
  try {
    const at::Tensor out = at::empty({B, H, T, D}, keys->options().requires_grad(false)), ws = bytes(need, *keys);
    x.q = q->const_data_ptr();
    x.k_new = k->const_data_ptr();
    x.v_new = v->const_data_ptr();
    x.out = out.mutable_data_ptr();
    const int rc = address<SharedFn>(args[0])(layout, address<const logkv_state_t*>(args[3]), prefix, &x,
                                              ws.mutable_data_ptr(), need, c10::cuda::getCurrentCUDAStream().stream());
    return rc ? failed(rc) : THPVariable_Wrap(out);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

void rotate_part(logkv_rotate_part_t& p, const at::Tensor& src, const at::Tensor* rotated, const at::Tensor* raw) {
  p.src = src.const_data_ptr();
  p.heads = (int32_t)src.size(1);
  p.rotate = rotated != nullptr;
  for (int i = 0; i < 3; ++i) p.src_strides[i] = src.stride(i);
  if (rotated) {
    p.rotated = rotated->mutable_data_ptr();
    for (int i = 0; i < 3; ++i) p.rotated_strides[i] = rotated->stride(i);
  }
  if (raw) {
    p.raw = raw->mutable_data_ptr();
    for (int i = 0; i < 3; ++i) p.raw_strides[i] = raw->stride(i);
  }
}

// Positions ([T] or [B, T] int32 or int64 on the device of `like`) into the arguments; false: not covered.
bool rotate_positions(logkv_rotate_args_t& a, PyObject* o, const at::Tensor& like) {
  if (o == Py_None) return true;
  const at::Tensor* p = tensor(o);
  if (!p || p->device() != like.device() || p->dim() < 1 || p->dim() > 2 || p->size(-1) != a.tokens ||
      (p->dim() == 2 && p->size(0) != a.batch) || (p->scalar_type() != at::kLong && p->scalar_type() != at::kInt))
    return false;
  a.positions = p->const_data_ptr();
  a.positions_wide = p->scalar_type() == at::kLong;
  a.position_strides[0] = p->dim() == 2 ? p->stride(0) : 0;
  a.position_strides[1] = p->stride(-1);
  return true;
}

int32_t dtype_code(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? LOGKV_DTYPE_F32 : LOGKV_DTYPE_BF16; }

// rotate(fn, rope, status, window keys, q, k, positions or None, pos0, interleaved): (q, k, raw keys), an error code, or
// None.  `window keys` [B, G, capacity, D] are the cache's.
PyObject* rotate(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 9) {
    PyErr_SetString(PyExc_TypeError, "rotate takes 9 arguments");
    return nullptr;
  }
  const at::Tensor *like = tensor(args[3]), *q = tensor(args[4]), *k = tensor(args[5]);
  if (!like || !q || !k || !like->is_cuda() || q->dim() != 4 || k->dim() != 4) Py_RETURN_NONE;
  const int64_t B = like->size(0), G = like->size(1), D = like->size(3), H = q->size(1), T = q->size(2);
  auto fits = [&](const at::Tensor& t, int64_t heads) {
    return t.size(0) == B && t.size(1) == heads && t.size(2) == T && t.size(3) == D && t.stride(3) == 1 &&
           t.scalar_type() == like->scalar_type() && t.device() == like->device() && !wants_gradient(t);
  };
  if (T < 1 || T > INT32_MAX || H < 1 || H % G || !fits(*q, H) || !fits(*k, G) ||
      c10::cuda::current_device() != like->get_device())
    Py_RETURN_NONE;
  logkv_rotate_args_t a{};
  a.n_parts = 2;
  a.batch = (int32_t)B;
  a.tokens = (int32_t)T;
  a.dim = (int32_t)D;
  a.dtype = dtype_code(*like);
  a.pos0 = PyLong_AsLongLong(args[7]);
  a.interleaved = PyObject_IsTrue(args[8]);
  a.status = address<int32_t*>(args[2]);
  if (PyErr_Occurred()) return nullptr;
  if (!rotate_positions(a, args[6], *like)) Py_RETURN_NONE;
  try {
    const auto opt = like->options().requires_grad(false);
    const at::Tensor qo = at::empty({B, H, T, D}, opt), ko = at::empty({B, G, T, D}, opt),
                     raw = a.interleaved ? at::empty({B, G, T, D}, opt) : *k;
    rotate_part(a.parts[0], *q, &qo, nullptr);
    rotate_part(a.parts[1], *k, &ko, a.interleaved ? &raw : nullptr);
    const int rc = address<RotateFn>(args[0])(address<const logkv_rope_t*>(args[1]), &a,
                                              c10::cuda::getCurrentCUDAStream().stream());
    if (rc) return failed(rc);
    if (a.interleaved) return Py_BuildValue("(NNN)", THPVariable_Wrap(qo), THPVariable_Wrap(ko), THPVariable_Wrap(raw));
    return Py_BuildValue("(NNO)", THPVariable_Wrap(qo), THPVariable_Wrap(ko), args[5]);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// append(fn, rope, status, row keys, raw keys, values, positions, ends, k, v, positions or None, ends [B, n] uint8 or
// None, pos0, first row, interleaved, q or None): 0 (the rotated q), an error code, or None.  The first five tensors
// take the rows: a cache's window, or a decoder's pending pair.
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 16) {
    PyErr_SetString(PyExc_TypeError, "append takes 16 arguments");
    return nullptr;
  }
  const at::Tensor* win[5];
  for (int i = 0; i < 5; ++i)
    if (!(win[i] = tensor(args[3 + i])) || !win[i]->is_cuda()) Py_RETURN_NONE;
  const at::Tensor *k = tensor(args[8]), *v = tensor(args[9]), *ends = tensor(args[11]), *q = tensor(args[15]);
  const at::Tensor& like = *win[0];
  if (!k || !v || (!ends && args[11] != Py_None) || (!q && args[15] != Py_None) || k->dim() != 4 || v->dim() != 4 ||
      (ends && ends->dim() != 2) || (q && q->dim() != 4))
    Py_RETURN_NONE;
  const int64_t B = like.size(0), G = like.size(1), C = like.size(2), D = like.size(3), T = k->size(2);
  const long long c0 = PyLong_AsLongLong(args[13]);
  auto fits = [&](const at::Tensor& t, int64_t heads) {
    return t.size(0) == B && t.size(1) == heads && t.size(2) == T && t.size(3) == D && t.stride(3) == 1 &&
           t.scalar_type() == like.scalar_type() && t.device() == like.device() && !wants_gradient(t);
  };
  logkv_rotate_args_t a{};
  a.n_parts = q ? 3 : 2;
  a.batch = (int32_t)B;
  a.tokens = (int32_t)T;
  a.dim = (int32_t)D;
  a.dtype = dtype_code(like);
  a.pos0 = PyLong_AsLongLong(args[12]);
  a.interleaved = PyObject_IsTrue(args[14]);
  a.status = address<int32_t*>(args[2]);
  if (PyErr_Occurred()) return nullptr;
  if (T < 1 || c0 < 0 || c0 + T > C || !fits(*k, G) || !fits(*v, G) ||
      (q && (q->size(1) < 1 || q->size(1) % G || !fits(*q, q->size(1)))) ||
      (ends && (ends->scalar_type() != at::kByte || ends->device() != like.device() || ends->size(0) != B ||
                ends->size(1) != T || (T > 1 && ends->stride(1) != 1))) ||
      c10::cuda::current_device() != like.get_device() || !rotate_positions(a, args[10], like))
    Py_RETURN_NONE;
  const int64_t offset = c0 * D * like.element_size();
  rotate_part(a.parts[0], *k, win[0], win[1]);
  rotate_part(a.parts[1], *v, nullptr, win[2]);
  a.parts[0].rotated = static_cast<char*>(a.parts[0].rotated) + offset;
  a.parts[0].raw = static_cast<char*>(a.parts[0].raw) + offset;
  a.parts[1].raw = static_cast<char*>(a.parts[1].raw) + offset;
  a.positions_out = static_cast<int64_t*>(win[3]->mutable_data_ptr()) + c0;
  a.positions_out_stride = win[3]->stride(0);
  if (ends) {
    a.ends = static_cast<const uint8_t*>(ends->const_data_ptr());
    a.ends_stride = ends->stride(0);
    a.ends_out = static_cast<uint8_t*>(win[4]->mutable_data_ptr()) + c0;
    a.ends_out_stride = win[4]->stride(0);
  }
  try {
    at::Tensor out;
    if (q) {
      out = at::empty({B, q->size(1), T, D}, like.options().requires_grad(false));
      rotate_part(a.parts[2], *q, &out, nullptr);
    }
    const int rc = address<RotateFn>(args[0])(address<const logkv_rope_t*>(args[1]), &a,
                                              c10::cuda::getCurrentCUDAStream().stream());
    return rc || !q ? failed(rc) : THPVariable_Wrap(out);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// A row's number: a Python number for all rows, or a contiguous [lead] tensor of `type`.
struct PerRow {
  const void* rows = nullptr;
  double value = 0;
  bool wide = false;
};
bool per_row(PyObject* o, const at::Tensor& x, bool whole, PerRow& out) {
  if (PyFloat_Check(o) || PyLong_Check(o)) {
    if (whole && !PyLong_Check(o)) return false;
    out.value = PyFloat_AsDouble(o);
    return in_range();
  }
  const at::Tensor* t = tensor(o);
  if (!t || t->dim() != x.dim() - 1 || t->device() != x.device() || !t->is_contiguous() ||
      !t->sizes().equals(x.sizes().slice(0, x.dim() - 1)) || wants_gradient(*t))
    return false;
  out.wide = t->scalar_type() == at::kLong;
  if (whole ? !out.wide && t->scalar_type() != at::kInt : t->scalar_type() != at::kFloat) return false;
  out.rows = t->const_data_ptr();
  return out.rows != nullptr;
}

// Entries of every row of x: [*lead, n] with the entries next to each other and evenly strided rows, or [n] for all.
bool entries(const at::Tensor* t, const at::Tensor& x, bool shared, int64_t& count, int64_t& stride) {
  if (!t || t->device() != x.device() || wants_gradient(*t)) return false;
  count = t->dim() ? t->size(-1) : 0;
  if (count < 1 || count > INT32_MAX || (count > 1 && t->stride(-1) != 1)) return false;
  stride = 0;
  if (shared && t->dim() == 1) return true;
  if (t->dim() != x.dim() || !t->sizes().slice(0, x.dim() - 1).equals(x.sizes().slice(0, x.dim() - 1))) return false;
  stride = t->stride(-2);
  return x.dim() == 2 || t->size(0) == 1 || t->stride(0) == stride * t->size(1);
}

// logits(fn, logits, history, lengths, prompt, repetition, presence, frequency, bias tokens, bias values, mask):
// adjusted logits, an error code, or None.  Tensors, numbers, or None.
PyObject* logits(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 11) {
    PyErr_SetString(PyExc_TypeError, "logits takes 11 arguments");
    return nullptr;
  }
  const at::Tensor* x = tensor(args[1]);
  if (!x || !x->is_cuda() || x->dim() < 2 || x->dim() > 3 || wants_gradient(*x) ||
      (x->scalar_type() != at::kFloat && x->scalar_type() != at::kBFloat16) ||
      c10::cuda::current_device() != x->get_device())
    Py_RETURN_NONE;
  const int64_t V = x->size(-1), W = x->size(-2), rows = x->dim() == 3 ? x->size(0) * W : W;
  if (V < 1 || V > (1 << 30) || rows < 1 || rows > 65535 || (V > 1 && x->stride(-1) != 1)) Py_RETURN_NONE;
  logkv_logits_args_t a{};
  PerRow len, pro, rep, pre, fre;
  if (!per_row(args[5], *x, false, rep) || !per_row(args[6], *x, false, pre) || !per_row(args[7], *x, false, fre))
    Py_RETURN_NONE;
  a.repetition = rep.rows ? 1.f : (float)rep.value;
  a.presence = (float)pre.value;
  a.frequency = (float)fre.value;
  if (!(a.repetition > 0.f && a.repetition < INFINITY) || !(a.presence - a.presence == 0.f) ||
      !(a.frequency - a.frequency == 0.f))
    Py_RETURN_NONE;
  a.repetitions = static_cast<const float*>(rep.rows);
  a.presences = static_cast<const float*>(pre.rows);
  a.frequencies = static_cast<const float*>(fre.rows);
  int64_t count = 0;
  if (args[2] != Py_None) {
    const at::Tensor* h = tensor(args[2]);
    if (!entries(h, *x, false, count, a.history_stride) || count > (1 << 30) ||
        (h->scalar_type() != at::kLong && h->scalar_type() != at::kInt) || !per_row(args[4], *x, true, pro))
      Py_RETURN_NONE;
    len.value = (double)count;
    if (args[3] != Py_None && !per_row(args[3], *x, true, len)) Py_RETURN_NONE;
    if (len.value < 0 || len.value > (double)count || pro.value < 0) Py_RETURN_NONE;
    a.history = h->const_data_ptr();
    a.history_wide = h->scalar_type() == at::kLong;
    a.history_len = (int32_t)count;
    a.length = (int32_t)len.value;
    a.prompt = (int32_t)(pro.value < (double)count ? pro.value : (double)count);
    a.lengths = len.rows;
    a.lengths_wide = len.wide;
    a.prompts = pro.rows;
    a.prompts_wide = pro.wide;
  } else if (args[3] != Py_None) {
    Py_RETURN_NONE;
  }
  if (args[8] != Py_None) {
    const at::Tensor *t = tensor(args[8]), *v = tensor(args[9]);
    int64_t values = 0;
    if (!entries(t, *x, true, count, a.bias_tokens_stride) || !entries(v, *x, true, values, a.bias_values_stride) ||
        values != count || t->dim() != v->dim() || count > LOGKV_LOGITS_MAX_BIAS || v->scalar_type() != at::kFloat ||
        (t->scalar_type() != at::kLong && t->scalar_type() != at::kInt))
      Py_RETURN_NONE;
    a.bias_tokens = t->const_data_ptr();
    a.bias_wide = t->scalar_type() == at::kLong;
    a.bias_values = static_cast<const float*>(v->const_data_ptr());
    a.bias_count = (int32_t)count;
  }
  if (args[10] != Py_None) {
    const at::Tensor* m = tensor(args[10]);
    if (!entries(m, *x, true, count, a.mask_stride) || count != (V + 31) / 32 || m->scalar_type() != at::kInt)
      Py_RETURN_NONE;
    a.mask = static_cast<const int32_t*>(m->const_data_ptr());
  }
  try {
    const at::Tensor out = at::empty(x->sizes(), x->options().requires_grad(false));
    a.logits = x->const_data_ptr();
    a.out = out.mutable_data_ptr();
    a.w_stride = x->stride(-2);
    a.out_w_stride = V;
    a.n_stride = x->dim() == 3 ? x->stride(0) : 0;
    a.out_n_stride = x->dim() == 3 ? W * V : 0;
    a.dtype = dtype_code(*x);
    a.rows = (int32_t)rows;
    a.width = (int32_t)W;
    a.vocab = (int32_t)V;
    const int rc = address<LogitsFn>(args[0])(&a, c10::cuda::getCurrentCUDAStream().stream());
    return rc ? failed(rc) : THPVariable_Wrap(out);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// A call with every C++ exception turned into a Python one (a tensor without strides throws where it is looked at).
using Call = PyObject* (*)(PyObject*, PyObject* const*, Py_ssize_t);
template <Call F>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  try {
    return F(self, args, n);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

#define LOGKV_METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<name>)), METH_FASTCALL, nullptr}

PyMethodDef methods[] = {
    LOGKV_METHOD(tree),   LOGKV_METHOD(beam),   LOGKV_METHOD(shared),
    LOGKV_METHOD(rotate), LOGKV_METHOD(append), LOGKV_METHOD(logits),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
