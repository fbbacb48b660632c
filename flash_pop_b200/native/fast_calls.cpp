// The host side of the operator calls, natively: argument checks, allocation of the results and of scratch memory, and the
// call into the C ABI.  In Python the same steps cost 50 to 65 us a call (measured), several times what most kernels of
// small and medium calls take.
//
// Every function here takes the ordinary call only - strided CUDA tensors of exactly torch.Tensor or Parameter type with the
// dtypes, shapes and strides the kernels read in place, no dispatch mode - and returns None for anything else, errors
// included; the caller then goes through the Python path, which copies, converts or raises.  A nonzero status of the C ABI
// comes back as an int.  Nothing is kept between calls but the addresses of the C ABI's entry points.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/core/TensorBody.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "../../include/flash_pop_b200.h"

namespace {

struct Entry {
  decltype(&fpb_retention_fwd) retention_fwd;
  decltype(&fpb_retention_bwd) retention_bwd;
  decltype(&fpb_pop_retention_fwd) pop_fwd;
  decltype(&fpb_pop_retention_bwd) pop_bwd;
  decltype(&fpb_pop_suffix_fwd) suffix_fwd;
  decltype(&fpb_pop_suffix_bwd) suffix_bwd;
  decltype(&fpb_retention_step) step;
  decltype(&fpb_workspace_bytes) workspace_bytes;
  decltype(&fpb_rotary) rotary;
  decltype(&fpb_groupnorm_gate_fwd) gate_fwd;
  decltype(&fpb_groupnorm_gate_bwd) gate_bwd;
  decltype(&fpb_layernorm_fwd) norm_fwd;
  decltype(&fpb_layernorm_bwd) norm_bwd;
  decltype(&fpb_column_sums) column_sums;
  decltype(&fpb_qk_norm_rotary_fwd) qk_norm_fwd;
  decltype(&fpb_qk_norm_rotary_bwd) qk_norm_bwd;
  decltype(&fpb_dropout) dropout;
  decltype(&fpb_embedding_fwd) embedding_fwd;
  decltype(&fpb_embedding_workspace) embedding_workspace;
  decltype(&fpb_embedding_bwd) embedding_bwd;
  decltype(&fpb_token_scores_fwd) scores_fwd;
  decltype(&fpb_token_scores_bwd) scores_bwd;
  decltype(&fpb_strerror) strerror;
} entry;
constexpr int ENTRIES = sizeof(Entry) / sizeof(void*), MAX_HEADS = 256;

struct NotOurs {};                               // thrown where a call is left to the Python path
#define NEED(cond) do { if (!(cond)) throw NotOurs{}; } while (0)

// A tensor the kernels may read through its address: exact type, strided CUDA memory, no lazy negation or conjugation.
at::Tensor tensor(PyObject* o) {
  NEED(THPVariable_CheckExact(o));
  const at::Tensor& t = THPVariable_Unpack(o);
  NEED(t.defined() && t.is_cuda() && t.layout() == at::kStrided && t.has_storage() && !t.is_neg() && !t.is_conj() && t.numel() > 0);
  return t;
}
at::Tensor maybe(PyObject* o) { return o == Py_None ? at::Tensor() : tensor(o); }
bool real(at::ScalarType t) { return t == at::kBFloat16 || t == at::kFloat; }
int32_t code(at::ScalarType t) { return t == at::kFloat ? FPB_F32 : FPB_BF16; }

// unit inner stride, and no row folded onto another (as _lib.unit_inner)
bool in_place(const at::Tensor& t) {
  const int n = (int)t.dim();
  if (t.is_contiguous()) return true;
  if (n == 0 || n > 6 || (t.stride(n - 1) != 1 && t.size(n - 1) != 1)) return false;
  int64_t st[6], sz[6];
  int m = 0;
  for (int i = 0; i < n - 1; ++i) {
    if (t.size(i) <= 1) continue;
    int j = m++;
    for (; j > 0 && st[j - 1] > t.stride(i); --j) { st[j] = st[j - 1]; sz[j] = sz[j - 1]; }
    st[j] = t.stride(i); sz[j] = t.size(i);
  }
  int64_t span = t.size(n - 1);
  for (int i = 0; i < m; ++i) {
    if (st[i] < span) return false;
    span = st[i] * sz[i];
  }
  return true;
}
bool aligned(const at::Tensor& t, int64_t bytes) {
  const int64_t vec = bytes / t.element_size();
  if ((uintptr_t)t.data_ptr() % bytes) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.stride(i) % vec) return false;
  return t.stride(t.dim() - 1) == 1;
}
bool state_ok(const at::Tensor& s) { return (s.stride(3) == 1 || s.size(3) == 1) && (s.stride(2) == s.size(3) || s.size(2) == 1); }

fpb_seq seq(const at::Tensor& t) {
  if (!t.defined()) return {nullptr, 0, 0, 0};
  return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}
fpb_seq seq3(const at::Tensor& t) { return {t.data_ptr(), t.stride(0), 0, t.stride(1)}; }      // (B, H, d): one token
fpb_state state(const at::Tensor& t) {
  if (!t.defined()) return {nullptr, 0, 0};
  return {t.data_ptr(), t.stride(0), t.stride(1)};
}

struct Decays {
  double g[MAX_HEADS];
  Decays(PyObject* o, int64_t heads) {
    NEED(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == heads && heads <= MAX_HEADS);
    for (int64_t h = 0; h < heads; ++h) {
      PyObject* f = PyTuple_GET_ITEM(o, h);
      NEED(PyFloat_Check(f));
      g[h] = PyFloat_AS_DOUBLE(f);
    }
  }
};

// (the allocator without the dispatcher, which adds half a microsecond; what has modes or a trace to tell of it was declined before)
at::Tensor make(at::IntArrayRef shape, const at::Tensor& like, at::ScalarType t) {
  return at::Tensor(at::detail::empty_cuda(shape, t, like.device(), std::nullopt));
}
at::Tensor make_like(const at::Tensor& t) { return at::empty_like(t, t.options().requires_grad(false)); }

// a call on t's device and its current stream
struct Place {
  c10::cuda::CUDAGuard guard;
  fpb_stream_t stream;
  explicit Place(const at::Tensor& t) : guard(t.device()), stream((fpb_stream_t)c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

struct Dims {
  fpb_dims d{};
  at::Tensor scratch;
  Dims(const at::Tensor& q, int64_t T, int64_t H, int64_t dk, int64_t dv, const Decays& g, int64_t block, int64_t flags, int64_t batch) {
    d.dtype = code(q.scalar_type()); d.B = (int32_t)batch; d.T = (int32_t)T; d.H = (int32_t)H; d.dk = (int32_t)dk; d.dv = (int32_t)dv;
    d.block_size = (int32_t)block; d.flags = (int32_t)flags; d.head_decays = g.g;
  }
  void with_scratch(const at::Tensor& q) {
    const int64_t need = entry.workspace_bytes(&d);
    if (need > 0) {
      scratch = at::empty({need}, q.options().dtype(at::kByte).requires_grad(false));
      d.workspace = scratch.data_ptr(); d.workspace_bytes = need;
    }
  }
};

at::ScalarType state_dtype(PyObject* asked, const at::Tensor& q, const at::Tensor& s) {
  at::ScalarType t = s.defined() ? s.scalar_type() : q.scalar_type();
  if (asked != Py_None) {
    NEED(THPDtype_Check(asked));
    t = reinterpret_cast<THPDtype*>(asked)->scalar_type;
  }
  NEED(t == q.scalar_type() || (t == at::kFloat && q.scalar_type() == at::kBFloat16));
  return t;
}

int64_t integer(PyObject* o) {
  NEED(PyLong_Check(o));
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) { PyErr_Clear(); throw NotOurs{}; }
  return v;
}
PyObject* wrap(const at::Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
PyObject* tuple_of(std::initializer_list<at::Tensor> ts) {
  PyObject* r = PyTuple_New((Py_ssize_t)ts.size());
  if (!r) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) {
    PyObject* o = wrap(t);
    if (!o) { Py_DECREF(r); return nullptr; }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

template <typename F> int unlocked(F f) {
  int r;
  Py_BEGIN_ALLOW_THREADS
  r = f();
  Py_END_ALLOW_THREADS
  return r;
}
// body with the exceptions of this file and of ATen turned into Python's
template <typename F> PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F body) {
  if (got != want) { PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got); return nullptr; }
  try {
    // (a trace would record the results' allocation and nothing that fills them; an autograd.Function it records as a whole)
    if (!entry.step || c10::impl::TorchDispatchModeTLS::any_modes_set() || torch::jit::tracer::isTracing()) Py_RETURN_NONE;
    return body();
  } catch (const NotOurs&) {
    Py_RETURN_NONE;
  } catch (const c10::OutOfMemoryError& e) {
    // (the Python path raises the allocator's own exception type with its message)
    Py_RETURN_NONE;
  } catch (python_error& e) {
    e.restore();                                 // (a saved-tensor hook's own)
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

void check_qkv(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& s) {
  NEED(q.dim() == 4 && v.dim() == 4 && k.sizes() == q.sizes() && v.size(0) == q.size(0) && v.size(1) == q.size(1) && v.size(2) == q.size(2));
  NEED(real(q.scalar_type()) && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type());
  NEED(k.device() == q.device() && v.device() == q.device() && in_place(q) && in_place(k) && in_place(v));
  if (s.defined())
    NEED(s.dim() == 4 && s.size(0) == q.size(0) && s.size(1) == q.size(2) && s.size(2) == q.size(3) && s.size(3) == v.size(3) &&
         s.device() == q.device() && state_ok(s));
}

// step(q, k, v, decays, prev_state, state_dtype, in_place) -> (o, state)
PyObject* step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    const at::Tensor q = tensor(a[0]), k = tensor(a[1]), v = tensor(a[2]), prev = maybe(a[4]);
    NEED(q.dim() == 3 && v.dim() == 3 && k.sizes() == q.sizes() && v.size(0) == q.size(0) && v.size(1) == q.size(1));
    NEED(real(q.scalar_type()) && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type());
    NEED(k.device() == q.device() && v.device() == q.device() && in_place(q) && in_place(k) && in_place(v));
    const int64_t B = q.size(0), H = q.size(1), dk = q.size(2), dv = v.size(2);
    const Decays g(a[3], H);
    at::ScalarType sdt = prev.defined() ? prev.scalar_type() : q.scalar_type();
    if (a[5] != Py_None) { NEED(THPDtype_Check(a[5])); sdt = reinterpret_cast<THPDtype*>(a[5])->scalar_type; }
    NEED(real(sdt));
    if (prev.defined())
      NEED(prev.dim() == 4 && prev.size(0) == B && prev.size(1) == H && prev.size(2) == dk && prev.size(3) == dv && prev.scalar_type() == sdt &&
           prev.device() == q.device() && state_ok(prev));
    const bool reuse = prev.defined() && a[6] == Py_True;
    Place here(q);
    const at::Tensor o = make({B, H, dv}, q, q.scalar_type()), out = reuse ? prev : make({B, H, dk, dv}, q, sdt);
    const Dims d(q, 1, H, dk, dv, g, 0, 0, B);
    const fpb_seq sq = seq3(q), sk = seq3(k), sv = seq3(v), so = seq3(o);
    const fpb_state s0 = state(prev), s1 = state(out);
    const int r = unlocked([&] { return entry.step(&d.d, code(sdt), &sq, &sk, &sv, &s0, &so, &s1, here.stream); });
    if (r) return PyLong_FromLong(r);
    PyObject* po = wrap(o);
    PyObject* ps = reuse ? Py_NewRef(a[4]) : wrap(out);
    return po && ps ? Py_BuildValue("(NN)", po, ps) : nullptr;
  });
}

// forward(q, k, v, s, decays, state_dtype, flags, block_size) -> (o, s_out) or, with block_size > 0, (o, block_states)
PyObject* forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const at::Tensor q = tensor(a[0]), k = tensor(a[1]), v = tensor(a[2]), s = maybe(a[3]);
    check_qkv(q, k, v, s);
    const int64_t B = q.size(0), T = q.size(1), H = q.size(2), dk = q.size(3), dv = v.size(3);
    const Decays g(a[4], H);
    const at::ScalarType sdt = state_dtype(a[5], q, s);
    NEED(!s.defined() || s.scalar_type() == sdt);
    const int64_t block = integer(a[7]), flags = integer(a[6]) | (sdt != q.scalar_type() ? FPB_FLAG_STATE_F32 : 0);
    NEED(block >= 0 && block <= INT32_MAX);
    Place here(q);
    const at::Tensor o = make({B, T, H, dv}, q, q.scalar_type());
    const at::Tensor end = block ? make({B, T / block, H, dk, dv}, q, sdt) : make({B, H, dk, dv}, q, sdt);
    Dims d(q, T, H, dk, dv, g, block, flags, B);
    d.with_scratch(q);
    const fpb_seq sq = seq(q), sk = seq(k), sv = seq(v), so = seq(o);
    const fpb_state s0 = state(s), s1 = block ? fpb_state{nullptr, 0, 0} : state(end);
    void* blocks = block && end.numel() > 0 ? end.data_ptr() : nullptr;
    const int r = unlocked([&] {
      return block ? entry.pop_fwd(&d.d, &sq, &sk, &sv, &s0, &so, blocks, here.stream)
                   : entry.retention_fwd(&d.d, &sq, &sk, &sv, &s0, &so, &s1, here.stream);
    });
    return r ? PyLong_FromLong(r) : tuple_of({o, end});
  });
}

// backward(q, k, v, s, dO, d_end, decays, state_dtype, flags, block_size, need_q, need_kv, need_s) -> (dQ, dK, dV, dS)
PyObject* backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 13, [&]() -> PyObject* {
    const at::Tensor q = tensor(a[0]), k = tensor(a[1]), v = tensor(a[2]), s = maybe(a[3]), dO = tensor(a[4]), dE = maybe(a[5]);
    check_qkv(q, k, v, s);
    const int64_t B = q.size(0), T = q.size(1), H = q.size(2), dk = q.size(3), dv = v.size(3);
    const Decays g(a[6], H);
    NEED(THPDtype_Check(a[7]));
    const at::ScalarType sdt = reinterpret_cast<THPDtype*>(a[7])->scalar_type;
    const int64_t block = integer(a[9]);
    const bool need_q = a[10] == Py_True, need_kv = a[11] == Py_True, need_s = a[12] == Py_True;
    NEED((need_q || need_kv) && block >= 0 && block <= INT32_MAX);
    NEED(dO.sizes() == v.sizes() && dO.scalar_type() == q.scalar_type() && dO.device() == q.device() && in_place(dO));
    if (dE.defined()) {
      NEED(dE.scalar_type() == sdt && dE.device() == q.device());
      if (block) NEED(dE.is_contiguous() && dE.dim() == 5 && dE.size(0) == B && dE.size(1) == T / block && dE.size(2) == H && dE.size(3) == dk && dE.size(4) == dv);
      else NEED(dE.dim() == 4 && dE.size(0) == B && dE.size(1) == H && dE.size(2) == dk && dE.size(3) == dv && state_ok(dE) &&
                (B == 1 || dE.stride(0) >= dk * dv) && (H == 1 || dE.stride(1) >= dk * dv));
    }
    const int64_t flags = integer(a[8]) | (need_q ? 0 : FPB_FLAG_SKIP_DQ) | (need_kv ? 0 : FPB_FLAG_SKIP_DKDV);
    Place here(q);
    const at::Tensor dQ = need_q ? make_like(q) : at::Tensor(), dK = need_kv ? make_like(k) : at::Tensor(),
                     dV = need_kv ? make_like(v) : at::Tensor(), dS = need_s ? make({B, H, dk, dv}, q, sdt) : at::Tensor();
    Dims d(q, T, H, dk, dv, g, block, flags, B);
    d.with_scratch(q);
    const fpb_seq sq = seq(q), sk = seq(k), sv = seq(v), so = seq(dO), gq = seq(dQ), gk = seq(dK), gv = seq(dV);
    const fpb_state s0 = state(s), s1 = block ? fpb_state{nullptr, 0, 0} : state(dE), gs = state(dS);
    const int r = unlocked([&] {
      return block ? entry.pop_bwd(&d.d, &sq, &sk, &sv, &s0, &so, dE.defined() ? dE.data_ptr() : nullptr, &gq, &gk, &gv, &gs, here.stream)
                   : entry.retention_bwd(&d.d, &sq, &sk, &sv, &s0, &so, &s1, &gq, &gk, &gv, &gs, here.stream);
    });
    return r ? PyLong_FromLong(r) : tuple_of({dQ, dK, dV, dS});
  });
}

// (B, M, P, H, d) as (B M, P, H, d) in place
at::Tensor rows_of(const at::Tensor& t) {
  NEED(t.dim() == 5 && (t.size(0) == 1 || t.size(1) == 1 || t.stride(0) == t.size(1) * t.stride(1)));
  const at::Tensor f = t.flatten(0, 1);
  NEED(f.data_ptr() == t.data_ptr() && in_place(f));
  return f;
}

// suffix_forward(sq, sk, sv, s, block_states, decays, flags) -> (o, fq, fk, fv)
PyObject* suffix_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    const at::Tensor sq = tensor(a[0]), sk = tensor(a[1]), sv = tensor(a[2]), s = maybe(a[3]), bs = tensor(a[4]);
    NEED(sq.dim() == 5 && sv.dim() == 5 && sk.sizes() == sq.sizes() && sv.sizes().slice(0, 4) == sq.sizes().slice(0, 4));
    const int64_t B = sq.size(0), M = sq.size(1), P = sq.size(2), H = sq.size(3), dk = sq.size(4), dv = sv.size(4);
    const at::ScalarType sdt = bs.scalar_type();
    NEED(real(sq.scalar_type()) && sk.scalar_type() == sq.scalar_type() && sv.scalar_type() == sq.scalar_type() &&
         (sdt == sq.scalar_type() || (sdt == at::kFloat && sq.scalar_type() == at::kBFloat16)));
    NEED(sk.device() == sq.device() && sv.device() == sq.device() && bs.device() == sq.device() && bs.dim() == 5 && bs.is_contiguous());
    NEED(bs.size(0) == B && M <= bs.size(1) + 1 && bs.size(2) == H && bs.size(3) == dk && bs.size(4) == dv && B * M <= INT32_MAX);
    if (s.defined())
      NEED(s.dim() == 4 && s.size(0) == B && s.size(1) == H && s.size(2) == dk && s.size(3) == dv && s.scalar_type() == sdt &&
           s.device() == sq.device() && state_ok(s));
    const Decays g(a[5], H);
    const at::Tensor fq = rows_of(sq), fk = rows_of(sk), fv = rows_of(sv);
    const int64_t flags = integer(a[6]) | (sdt != sq.scalar_type() ? FPB_FLAG_STATE_F32 : 0);
    Place here(fq);
    const at::Tensor o = make({B, M, P, H, dv}, sq, sq.scalar_type());
    const Dims d(fq, P, H, dk, dv, g, 0, flags, B);
    const fpb_seq q4 = seq(fq), k4 = seq(fk), v4 = seq(fv), o4{o.data_ptr(), P * H * dv, H * dv, dv};
    const fpb_state s0 = state(s);
    const int r = unlocked([&] {
      return entry.suffix_fwd(&d.d, (int32_t)M, (int32_t)bs.size(1), &q4, &k4, &v4, &s0, bs.data_ptr(), &o4, here.stream);
    });
    return r ? PyLong_FromLong(r) : tuple_of({o, fq, fk, fv});
  });
}

// suffix_backward(fq, fk, fv, s, block_states, dO (B, M, P, H, dv), decays, flags) -> (dQ, dK, dV (B, M, P, H, d), dS, d_block_states)
PyObject* suffix_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const at::Tensor fq = tensor(a[0]), fk = tensor(a[1]), fv = tensor(a[2]), s = maybe(a[3]), bs = tensor(a[4]), dO5 = tensor(a[5]);
    NEED(dO5.dim() == 5 && dO5.scalar_type() == fq.scalar_type() && dO5.device() == fq.device());
    const int64_t B = dO5.size(0), M = dO5.size(1), P = fq.size(1), H = fq.size(2), dk = fq.size(3), dv = fv.size(3);
    NEED(B * M == fq.size(0) && dO5.size(2) == P && dO5.size(3) == H && dO5.size(4) == dv);
    const at::Tensor dO = rows_of(dO5);
    NEED(fk.sizes() == fq.sizes() && fv.dim() == 4 && fk.scalar_type() == fq.scalar_type() && fv.scalar_type() == fq.scalar_type() && bs.dim() == 5 &&
         bs.is_contiguous() && bs.device() == fq.device() && in_place(fq) && in_place(fk) && in_place(fv) && (!s.defined() || state_ok(s)));
    const Decays g(a[6], H);
    Place here(fq);
    const at::Tensor dQ = make_like(fq), dK = make_like(fk), dV = make_like(fv), dB = make_like(bs),
                     dS = s.defined() ? make({B, H, dk, dv}, fq, bs.scalar_type()) : at::Tensor();
    const Dims d(fq, P, H, dk, dv, g, 0, integer(a[7]), B);
    const fpb_seq q4 = seq(fq), k4 = seq(fk), v4 = seq(fv), o4 = seq(dO), gq = seq(dQ), gk = seq(dK), gv = seq(dV);
    const fpb_state s0 = state(s), gs = state(dS);
    const int r = unlocked([&] {
      return entry.suffix_bwd(&d.d, (int32_t)M, (int32_t)bs.size(1), &q4, &k4, &v4, &s0, bs.data_ptr(), &o4, &gq, &gk, &gv, &gs,
                              dB.data_ptr(), here.stream);
    });
    if (r) return PyLong_FromLong(r);
    auto rows = [&](const at::Tensor& t) { return t.unflatten(0, {B, M}); };
    return tuple_of({rows(dQ), rows(dK), rows(dV), dS, dB});
  });
}

// rotary(q, k, phasors, conjugate, out_dtype) -> (q', k')
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    const at::Tensor q = tensor(a[0]), k = tensor(a[1]), ph = tensor(a[2]);
    NEED(q.dim() == 4 && k.sizes() == q.sizes() && real(q.scalar_type()) && k.scalar_type() == q.scalar_type() && k.device() == q.device());
    const int64_t B = q.size(0), T = q.size(1), H = q.size(2), d = q.size(3);
    NEED(d % 8 == 0 && ph.scalar_type() == at::kFloat && ph.is_contiguous() && ph.dim() == 4 && (ph.size(0) == 1 || ph.size(0) == B) &&
         ph.size(1) == T && ph.size(2) == d / 2 && ph.size(3) == 2 && ph.device() == q.device() && (uintptr_t)ph.data_ptr() % 16 == 0);
    NEED(THPDtype_Check(a[4]));
    const at::ScalarType odt = reinterpret_cast<THPDtype*>(a[4])->scalar_type;
    NEED(real(odt) && in_place(q) && in_place(k) && aligned(q, 16) && aligned(k, 16));
    Place here(q);
    const at::Tensor q2 = make({B, T, H, d}, q, odt), k2 = make({B, T, H, d}, q, odt);
    const fpb_seq qi = seq(q), ki = seq(k), qo = seq(q2), ko = seq(k2);
    const int r = unlocked([&] {
      return entry.rotary((int32_t)B, (int32_t)T, (int32_t)H, (int32_t)d, code(q.scalar_type()), code(odt), a[3] == Py_True ? 1 : 0,
                          (const float*)ph.data_ptr(), ph.size(0) == 1 ? 0 : T * (d / 2), &qi, &ki, &qo, &ko, here.stream);
    });
    return r ? PyLong_FromLong(r) : tuple_of({q2, k2});
  });
}

void check_gate(const at::Tensor& o, const at::Tensor& z) {
  NEED(o.dim() == 4 && z.sizes() == o.sizes() && real(o.scalar_type()) && z.scalar_type() == o.scalar_type() && z.device() == o.device());
  const int64_t nb = o.scalar_type() == at::kFloat ? 8 : 4;
  NEED(in_place(o) && in_place(z) && aligned(o, nb) && aligned(z, nb));
}
// gate_forward(o, z, eps, swish) -> (y,)
PyObject* gate_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    const at::Tensor o = tensor(a[0]), z = tensor(a[1]);
    check_gate(o, z);
    NEED(PyFloat_Check(a[2]));
    Place here(o);
    const at::Tensor y = make(o.sizes(), o, o.scalar_type());
    const fpb_seq so = seq(o), sz = seq(z), sy = seq(y);
    const int r = unlocked([&] {
      return entry.gate_fwd((int32_t)o.size(0), (int32_t)o.size(1), (int32_t)o.size(2), (int32_t)o.size(3), code(o.scalar_type()),
                            (float)PyFloat_AS_DOUBLE(a[2]), a[3] == Py_True ? 1 : 0, &so, &sz, &sy, here.stream);
    });
    return r ? PyLong_FromLong(r) : tuple_of({y});
  });
}
// gate_backward(o, z, dy, eps, swish) -> (d_o, d_z)
PyObject* gate_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    const at::Tensor o = tensor(a[0]), z = tensor(a[1]), dy = tensor(a[2]);
    check_gate(o, z);
    check_gate(o, dy);
    NEED(PyFloat_Check(a[3]));
    Place here(o);
    const at::Tensor d_o = make(o.sizes(), o, o.scalar_type()), d_z = make(o.sizes(), o, o.scalar_type());
    const fpb_seq so = seq(o), sz = seq(z), sy = seq(dy), go = seq(d_o), gz = seq(d_z);
    const int r = unlocked([&] {
      return entry.gate_bwd((int32_t)o.size(0), (int32_t)o.size(1), (int32_t)o.size(2), (int32_t)o.size(3), code(o.scalar_type()),
                            (float)PyFloat_AS_DOUBLE(a[3]), a[4] == Py_True ? 1 : 0, &so, &sz, &sy, &go, &gz, here.stream);
    });
    return r ? PyLong_FromLong(r) : tuple_of({d_o, d_z});
  });
}

const float* param(const at::Tensor& t, int64_t d, const at::Tensor& like) {
  if (!t.defined()) return nullptr;
  NEED(t.scalar_type() == at::kFloat && t.is_contiguous() && t.dim() == 1 && t.size(0) == d && t.device() == like.device() &&
       (uintptr_t)t.data_ptr() % 16 == 0);
  return (const float*)t.data_ptr();
}
void check_norm(const at::Tensor& x) {
  NEED(x.dim() >= 1 && real(x.scalar_type()) && x.is_contiguous() && (uintptr_t)x.data_ptr() % 16 == 0);
  const int64_t vec = 16 / x.element_size(), d = x.size(-1);
  NEED(d % vec == 0 && d <= 128 * vec);
}
// norm_forward(x, weight, bias, eps) -> (y,)
PyObject* norm_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    const at::Tensor x = tensor(a[0]), w = maybe(a[1]), b = maybe(a[2]);
    check_norm(x);
    NEED(PyFloat_Check(a[3]));
    const int64_t d = x.size(-1), rows = x.numel() / d;
    const float *pw = param(w, d, x), *pb = param(b, d, x);
    Place here(x);
    const at::Tensor y = make(x.sizes(), x, x.scalar_type());
    const int r = unlocked([&] {
      return entry.norm_fwd(rows, (int32_t)d, code(x.scalar_type()), (float)PyFloat_AS_DOUBLE(a[3]), x.data_ptr(), d, pw, pb, y.data_ptr(), d,
                            here.stream);
    });
    return r ? PyLong_FromLong(r) : tuple_of({y});
  });
}
// norm_backward(x, weight, dy, eps, need_w, need_b) -> (dx, dw, db), the last two fp32
PyObject* norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&]() -> PyObject* {
    const at::Tensor x = tensor(a[0]), w = maybe(a[1]), dy = tensor(a[2]);
    check_norm(x);
    check_norm(dy);
    NEED(PyFloat_Check(a[3]) && dy.numel() == x.numel() && dy.size(-1) == x.size(-1) && dy.scalar_type() == x.scalar_type() && dy.device() == x.device());
    const int64_t d = x.size(-1), rows = x.numel() / d;
    const float* pw = param(w, d, x);
    Place here(x);
    const at::Tensor dx = make(dy.sizes(), x, x.scalar_type());
    const at::Tensor dw = a[4] == Py_True ? make({d}, x, at::kFloat) : at::Tensor(), db = a[5] == Py_True ? make({d}, x, at::kFloat) : at::Tensor();
    const int r = unlocked([&] {
      return entry.norm_bwd(rows, (int32_t)d, code(x.scalar_type()), (float)PyFloat_AS_DOUBLE(a[3]), x.data_ptr(), d, pw, dy.data_ptr(), d,
                            dx.data_ptr(), dw.defined() ? (float*)dw.data_ptr() : nullptr, db.defined() ? (float*)db.data_ptr() : nullptr, here.stream);
    });
    return r ? PyLong_FromLong(r) : tuple_of({dx, dw, db});
  });
}

// column_sums(g (..., n), a or None) -> (sums (n), d_a or None): all contiguous bf16
PyObject* column_sums(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 2, [&]() -> PyObject* {
    const at::Tensor g = tensor(a[0]), act = maybe(a[1]);
    NEED(g.scalar_type() == at::kBFloat16 && g.dim() >= 1 && g.is_contiguous() && g.size(-1) % 64 == 0 && (uintptr_t)g.data_ptr() % 16 == 0);
    if (act.defined())
      NEED(act.scalar_type() == at::kBFloat16 && act.is_contiguous() && act.sizes() == g.sizes() && act.device() == g.device() &&
           (uintptr_t)act.data_ptr() % 16 == 0);
    const int64_t cols = g.size(-1), rows = g.numel() / cols;
    NEED(cols <= FPB_COLUMN_SUMS_SCRATCH / 4);
    Place here(g);
    const at::Tensor scratch = make({FPB_COLUMN_SUMS_SCRATCH}, g, at::kByte);
    const at::Tensor sums = make({cols}, g, at::kBFloat16), d_a = act.defined() ? make(g.sizes(), g, at::kBFloat16) : at::Tensor();
    const int r = unlocked([&] {
      return entry.column_sums(rows, cols, g.data_ptr(), cols, act.defined() ? act.data_ptr() : nullptr, d_a.defined() ? d_a.data_ptr() : nullptr,
                               scratch.data_ptr(), sums.data_ptr(), here.stream);
    });
    return r ? PyLong_FromLong(r) : tuple_of({sums, d_a});
  });
}

// ---- operators with autograd nodes of their own ---------------------------------------------------------------------
// A small call's gradient through torch.autograd.Function costs 15 to 30 us of Python more than through these nodes.  The function that Python calls
// checks, and leaves to Python (NotOurs) what is not the ordinary call; `run` computes, alone or in a node where a gradient is
// recorded.  A backward takes whatever strides the gradients have, by copying them.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::vector<at::Tensor> Tensors;

struct Status { int code; };                     // thrown by `run`: a status of the C ABI
void ran(int status) { if (status) throw Status{status}; }
void ran_backward(int status) { TORCH_CHECK(status == 0, "flash_pop_b200: ", entry.strerror(status)); }

bool graph_wanted(std::initializer_list<at::Tensor> ts) {
  for (const at::Tensor& t : ts)
    if (t.defined()) NEED(!t._fw_grad(0).defined());             // (forward-mode gradients: Python says that there are none)
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
// body, with a status of the C ABI as an int
template <typename F> PyObject* guarded_call(Py_ssize_t got, Py_ssize_t want, F body) {
  return guarded(got, want, [&]() -> PyObject* {
    try {
      const Tensors out = body();
      PyObject* r = PyTuple_New((Py_ssize_t)out.size());
      for (size_t i = 0; r && i < out.size(); ++i) {
        PyObject* o = wrap(out[i]);
        if (!o) { Py_DECREF(r); return nullptr; }
        PyTuple_SET_ITEM(r, (Py_ssize_t)i, o);
      }
      return r;
    } catch (const Status& s) {
      return PyLong_FromLong(s.code);
    }
  });
}
// The node that runs, in a captured backward pass, hands no gradient to a node made on the default stream (a leaf's, while an eager
// graph of the leaf lives): the engine would make that stream wait within the capture, which is an error where nothing catches it.
void may_be_captured() {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const std::shared_ptr<torch::autograd::Node> node = torch::autograd::get_current_node();
  if (!node) return;
  for (size_t i = 0; i < node->num_outputs(); ++i) {
    const torch::autograd::Edge& to = node->next_edge(i);
    if (!to.is_valid() || !node->task_should_compute_output(i)) continue;
    const std::optional<c10::Stream> stream = to.function->stream();
    TORCH_CHECK(!stream || *stream != c10::cuda::getDefaultCUDAStream(stream->device_index()).unwrap(),
                "flash_pop_b200: this backward pass is being captured, and one of its gradients belongs to a graph made on the default stream, which no "
                "capture may touch: release the outputs of the eager calls with the same leaves first, or make them on the capture's stream");
  }
}
// What a backward returns where a graph of it is recorded: a second derivative raises.
variable_list once(variable_list out, bool graph) {
  if (!graph) return out;
  variable_list in;
  for (const at::Tensor& t : out) in.push_back(t.defined() ? t.detach().requires_grad_(true) : t);
  return torch::autograd::DelayedError("trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)in.size())
      .apply(std::move(in));
}
at::Tensor dense(const at::Tensor& t) {          // contiguous and 16-byte aligned
  const at::Tensor c = t.contiguous();
  return (uintptr_t)c.data_ptr() % 16 ? c.clone() : c;
}
at::Tensor readable(const at::Tensor& t) {       // rows as the kernels take them, copied if need be
  if (t.numel() == 0 || (in_place(t) && aligned(t, 16))) return t;
  const at::Tensor c = dense(t);                 // (contiguous as it was, it may keep a stride that no element uses)
  return aligned(c, 16) ? c : c.clone(at::MemoryFormat::Contiguous);
}
// (an absent tensor is no input of a node, nor counted among them)
typedef std::optional<at::Tensor> Maybe;
Maybe given(const at::Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }
at::Tensor or_none(const Maybe& t) { return t ? *t : at::Tensor(); }
double real_number(PyObject* o) {
  NEED(PyFloat_Check(o));
  return PyFloat_AS_DOUBLE(o);
}

// queries and keys (B, T, heads, d) with the weights (d, fp32) and phasors of their norm and rotation
struct QkNorm : torch::autograd::Function<QkNorm> {
  struct Call {
    at::Tensor q, k, wq, wk, ph;
    float eps;
    int32_t B, T, Hq, Hk, d;
    int64_t step = 0;
    Call(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& wq_, const at::Tensor& wk_, const at::Tensor& ph_, double eps_)
        : q(q_), k(k_), wq(wq_), wk(wk_), ph(ph_), eps((float)eps_) {
      B = (int32_t)q.size(0); T = (int32_t)q.size(1); Hq = (int32_t)q.size(2); Hk = (int32_t)k.size(2); d = (int32_t)q.size(3);
      if (ph.defined() && ph.size(0) > 1) step = (int64_t)T * (d / 2);
    }
    void check() const {
      NEED(real(q.scalar_type()) && k.scalar_type() == q.scalar_type() && k.device() == q.device() && k.size(0) == B && k.size(1) == T && k.size(3) == d);
      NEED(d % 8 == 0 && d <= 256 && eps >= 0.0f && q.numel() < INT32_MAX && k.numel() < INT32_MAX);
      NEED(in_place(q) && aligned(q, 16) && in_place(k) && aligned(k, 16));
      param(wq, d, q); param(wk, d, q);
      if (ph.defined())
        NEED(ph.dim() == 4 && (ph.size(0) == 1 || ph.size(0) == B) && ph.size(1) == T && ph.size(2) == d / 2 && ph.size(3) == 2 && ph.is_contiguous() &&
             ph.scalar_type() == at::kFloat && ph.device() == q.device() && (uintptr_t)ph.data_ptr() % 16 == 0);
    }
    static const float* data(const at::Tensor& t) { return t.defined() ? (const float*)t.data_ptr() : nullptr; }
  };
  static Tensors run(const Call& c) {
    Place here(c.q);
    const at::Tensor yq = make(c.q.sizes(), c.q, c.q.scalar_type()), yk = make(c.k.sizes(), c.q, c.q.scalar_type());
    const fpb_seq sq = seq(c.q), sk = seq(c.k), oq = seq(yq), ok = seq(yk);
    ran(unlocked([&] {
      return entry.qk_norm_fwd(c.B, c.T, c.Hq, c.Hk, c.d, code(c.q.scalar_type()), c.eps, c.data(c.wq), c.data(c.wk), c.data(c.ph), c.step, &sq, &sk, &oq,
                               &ok, here.stream);
    }));
    return {yq, yk};
  }
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const Maybe& wq, const Maybe& wk, const Maybe& ph,
                               double eps) {
    variable_list y = run(Call(q, k, or_none(wq), or_none(wk), or_none(ph), eps));
    ctx->save_for_backward({q, k, or_none(wq), or_none(wk), or_none(ph)});
    ctx->saved_data["eps"] = eps;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const bool graph = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    may_be_captured();
    const variable_list v = ctx->get_saved_variables();
    const Call c(v[0], v[1], v[2], v[3], v[4], ctx->saved_data["eps"].toDouble());
    Place here(c.q);
    const at::Tensor dyq = readable(g[0]), dyk = readable(g[1]);
    const at::Tensor dq = make(c.q.sizes(), c.q, c.q.scalar_type()), dk = make(c.k.sizes(), c.q, c.q.scalar_type()),
                     dwq = c.wq.defined() && ctx->needs_input_grad(2) ? make({c.d}, c.q, at::kFloat) : at::Tensor(),
                     dwk = c.wk.defined() && ctx->needs_input_grad(c.wq.defined() ? 3 : 2) ? make({c.d}, c.q, at::kFloat) : at::Tensor(),
                     scratch = make({FPB_QK_NORM_SCRATCH(c.d)}, c.q, at::kByte);
    const fpb_seq sq = seq(c.q), sk = seq(c.k), gq = seq(dyq), gk = seq(dyk), oq = seq(dq), ok = seq(dk);
    ran_backward(entry.qk_norm_bwd(c.B, c.T, c.Hq, c.Hk, c.d, code(c.q.scalar_type()), c.eps, c.data(c.wq), c.data(c.wk), c.data(c.ph), c.step, &sq, &sk,
                                   &gq, &gk, &oq, &ok, dwq.defined() ? (float*)dwq.data_ptr() : nullptr, dwk.defined() ? (float*)dwk.data_ptr() : nullptr,
                                   scratch.data_ptr(), here.stream));
    return once({dq, dk, dwq, dwk, at::Tensor(), at::Tensor()}, graph);
  }
};
// qk_norm_rotary(q, k, wq, wk, phasors, eps) -> (yq, yk)
PyObject* qk_norm_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded_call(n, 6, [&]() -> Tensors {
    const at::Tensor q = tensor(a[0]), k = tensor(a[1]), wq = maybe(a[2]), wk = maybe(a[3]), ph = maybe(a[4]);
    const double eps = real_number(a[5]);
    NEED(q.dim() == 4 && k.dim() == 4 && !(ph.defined() && ph.requires_grad()));
    const QkNorm::Call c(q, k, wq, wk, ph, eps);
    c.check();
    return graph_wanted({q, k, wq, wk}) ? QkNorm::apply(q, k, given(wq), given(wk), given(ph), eps) : QkNorm::run(c);
  });
}

struct Dropout : torch::autograd::Function<Dropout> {
  static at::Tensor run(const at::Tensor& x, const at::Tensor& res, double p, const at::Tensor& seed, bool backward) {
    Place here(x);
    const at::Tensor y = make(x.sizes(), x, x.scalar_type());
    auto call = [&] {
      return entry.dropout(x.numel(), code(x.scalar_type()), p, (const int64_t*)seed.data_ptr(), x.data_ptr(), res.defined() ? res.data_ptr() : nullptr,
                           y.data_ptr(), here.stream);
    };
    if (backward) ran_backward(call()); else ran(unlocked(call));
    return y;
  }
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const Maybe& res, double p, const at::Tensor& seed) {
    const at::Tensor y = run(x, or_none(res), p, seed, false);
    ctx->save_for_backward({seed});
    ctx->saved_data["residual"] = res.has_value();
    ctx->saved_data["p"] = p;
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const bool graph = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    may_be_captured();
    const at::Tensor seed = ctx->get_saved_variables()[0];
    const at::Tensor dx = ctx->needs_input_grad(0) ? run(dense(g[0]), at::Tensor(), ctx->saved_data["p"].toDouble(), seed, true) : at::Tensor();
    return once({dx, ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1) ? g[0] : at::Tensor(), at::Tensor(), at::Tensor()}, graph);
  }
};
// dropout(x, residual or None, p, seed) -> (y,)
PyObject* dropout(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded_call(n, 4, [&]() -> Tensors {
    const at::Tensor x = tensor(a[0]), res = maybe(a[1]), seed = tensor(a[3]);
    const double p = real_number(a[2]);
    NEED(real(x.scalar_type()) && x.is_contiguous() && p >= 0.0 && p <= 1.0);
    if (res.defined()) NEED(res.scalar_type() == x.scalar_type() && res.sizes() == x.sizes() && res.is_contiguous() && res.device() == x.device());
    NEED(seed.scalar_type() == at::kLong && seed.numel() == 1 && seed.device() == x.device());
    if (graph_wanted({x, res})) return Dropout::apply(x, given(res), p, seed);
    return {Dropout::run(x, res, p, seed, false)};
  });
}

int64_t pitch(const at::Tensor& t) {             // of a matrix whose rows can be read in place
  NEED(t.dim() == 2 && (t.stride(1) == 1 || t.size(1) == 1) && (t.size(0) == 1 || t.stride(0) >= t.size(1)));
  return t.size(0) > 1 ? t.stride(0) : t.size(1);
}
at::Tensor ids(PyObject* o, const at::Tensor& like) {
  const at::Tensor t = tensor(o);
  NEED(t.scalar_type() == at::kLong && t.is_contiguous() && t.device() == like.device());
  return t;
}
std::vector<int64_t> with_last(at::IntArrayRef sizes, int64_t last) {
  std::vector<int64_t> shape(sizes.begin(), sizes.end());
  shape.push_back(last);
  return shape;
}
at::Tensor embedding_rows(const at::Tensor& t, const at::Tensor& w, double scale) {
  const int64_t stride = pitch(w), D = w.size(1);
  Place here(w);
  const at::Tensor y = make(with_last(t.sizes(), D), w, w.scalar_type());
  ran(unlocked([&] {
    return entry.embedding_fwd(t.numel(), w.size(0), (int32_t)D, code(w.scalar_type()), (const int64_t*)t.data_ptr(), w.data_ptr(), stride, (float)scale,
                               y.data_ptr(), here.stream);
  }));
  return y;
}
at::Tensor embedding_gradient(const at::Tensor& t, const at::Tensor& g, int64_t V, double scale, int64_t padding) {
  const int64_t D = g.size(-1), N = t.numel();
  Place here(g);
  const at::Tensor dy = dense(g), dw = make({V, D}, dy, dy.scalar_type());
  const int64_t need = entry.embedding_workspace(N, V, (int32_t)D);
  const at::Tensor scratch = need > 16 ? make({need}, dy, at::kByte) : dw;         // (a few ids' is not touched)
  ran_backward(entry.embedding_bwd(N, V, (int32_t)D, code(dy.scalar_type()), (const int64_t*)t.data_ptr(), padding, (float)scale, dy.data_ptr(), D,
                                   dw.data_ptr(), scratch.data_ptr(), need, here.stream));
  return dw;
}
// The node as compiled autograd takes it: Function's, whose forward is called for its node alone and computes nothing.
struct CompiledEmbedding : torch::autograd::Function<CompiledEmbedding> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& t, const at::Tensor& w, double scale, int64_t padding) {
    ctx->save_for_backward({t});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["padding"] = padding;
    ctx->saved_data["V"] = w.size(0);
    return make(with_last(t.sizes(), w.size(1)), w, w.scalar_type());
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    at::NoGradGuard no_grad;
    return {at::Tensor(), embedding_gradient(ctx->get_saved_variables()[0], g[0], ctx->saved_data["V"].toInt(), ctx->saved_data["scale"].toDouble(),
                                             ctx->saved_data["padding"].toInt()), at::Tensor(), at::Tensor()};
  }
};
// A node without Function's context, whose making and running are 4 of the 55 us that a lookup and its gradient would take on the host.
struct Embedding : torch::autograd::Node {
  torch::autograd::SavedVariable tokens;
  double scale;
  int64_t padding, V, D;
  at::TensorOptions like;                        // of the table
  mutable std::shared_ptr<torch::autograd::Node> compiled;

  static at::Tensor run(const at::Tensor& t, const at::Tensor& w, double scale, int64_t padding) {
    at::Tensor y = embedding_rows(t, w, scale);
    const std::shared_ptr<Embedding> node(new Embedding(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(t, w));
    node->tokens = torch::autograd::SavedVariable(t, false);
    node->scale = scale; node->padding = padding; node->V = w.size(0); node->D = w.size(1);
    node->like = w.options().requires_grad(false);
    torch::autograd::set_history(y, node);
    return y;
  }
  std::string name() const override { return "EmbeddingBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    tokens.reset_data();
    compiled.reset();
  }
  variable_list apply(variable_list&& g) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const bool graph = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    may_be_captured();
    const at::Tensor t = tokens.unpack();        // (raises where it was freed or changed)
    return once({at::Tensor(), g[0].defined() ? embedding_gradient(t, g[0], V, scale, padding) : at::Tensor()}, graph);
  }
  void compiled_args(torch::dynamo::autograd::CompiledNodeArgs& args) const override {
    if (!compiled) {
      at::AutoGradMode grad(true);
      const at::Tensor w = at::empty({1, 1}, like).expand({V, D}).requires_grad_(true);       // (its shape counts)
      compiled = CompiledEmbedding::apply(tokens.unpack(), w, scale, padding).grad_fn();
    }
    compiled->compiled_args(args);
  }
  variable_list apply_with_saved(const variable_list& inputs, torch::dynamo::autograd::SwapSavedVariables& saved) override {
    return compiled->apply_with_saved(inputs, saved);
  }
};
// embedding(tokens, weight, scale, padding) -> (y,)
PyObject* embedding(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded_call(n, 4, [&]() -> Tensors {
    const at::Tensor w = tensor(a[1]), t = ids(a[0], w);
    const double scale = real_number(a[2]);
    const int64_t padding = integer(a[3]);
    NEED(real(w.scalar_type()) && w.dim() == 2 && w.size(1) <= 1 << 20);
    pitch(w);
    return {graph_wanted({w}) ? Embedding::run(t, w, scale, padding) : embedding_rows(t, w, scale)};
  });
}

struct Scores : torch::autograd::Function<Scores> {
  static int64_t stride(const at::Tensor& z) { return z.is_contiguous() ? z.size(-1) : pitch(z); }
  // logprob, entropy, top_logprob, top_tokens (undefined without alternatives), stats
  static Tensors run(const at::Tensor& z, const at::Tensor& t, int64_t top) {
    const int64_t V = z.size(-1), rows = t.numel(), pitch_z = stride(z);
    Place here(z);
    const at::Tensor lp = make(t.sizes(), z, at::kFloat), h = make(t.sizes(), z, at::kFloat), stats = make({rows, 2}, z, at::kFloat);
    at::Tensor tl, tt;
    if (top) { tl = make(with_last(t.sizes(), top), z, at::kFloat); tt = make(with_last(t.sizes(), top), z, at::kLong); }
    ran(unlocked([&] {
      return entry.scores_fwd(rows, (int32_t)V, code(z.scalar_type()), (int32_t)top, z.data_ptr(), pitch_z, (const int64_t*)t.data_ptr(), (float*)lp.data_ptr(),
                              (float*)h.data_ptr(), (float*)stats.data_ptr(), top ? (float*)tl.data_ptr() : nullptr,
                              top ? (int64_t*)tt.data_ptr() : nullptr, here.stream);
    }));
    return {lp, h, tl, tt, stats};
  }
  static variable_list forward(AutogradContext* ctx, const at::Tensor& z, const at::Tensor& t, int64_t top) {
    Tensors r = run(z, t, top);
    ctx->save_for_backward({z, t, r[1], r[4], r[3]});
    ctx->set_materialize_grads(false);
    if (top) ctx->mark_non_differentiable({r[3]});
    r.resize(top ? 4 : 2);
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const bool graph = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    may_be_captured();
    const variable_list v = ctx->get_saved_variables();
    const at::Tensor &z = v[0], &t = v[1], &tt = v[4];
    const int64_t V = z.size(-1), rows = t.numel(), top = tt.defined() ? tt.size(-1) : 0;
    at::Tensor gs[3];
    for (size_t i = 0; i < 3 && i < g.size(); ++i)
      if (g[i].defined()) gs[i] = g[i].contiguous();
    if (!gs[0].defined() && !gs[1].defined() && !gs[2].defined()) return {at::Tensor(), at::Tensor(), at::Tensor()};
    Place here(z);
    const at::Tensor d = make(z.sizes(), z, z.scalar_type());
    auto at = [](const at::Tensor& x) { return x.defined() ? (const float*)x.data_ptr() : nullptr; };
    ran_backward(entry.scores_bwd(rows, (int32_t)V, code(z.scalar_type()), (int32_t)top, z.data_ptr(), stride(z), (const int64_t*)t.data_ptr(), at(v[2]),
                                  at(v[3]), tt.defined() ? (const int64_t*)tt.data_ptr() : nullptr, at(gs[0]), at(gs[1]), at(gs[2]), d.data_ptr(), V,
                                  here.stream));
    return once({d, at::Tensor(), at::Tensor()}, graph);
  }
};
// token_scores(logits (..., V), tokens (...), top) -> (logprob, entropy, top_logprob or None, top_tokens or None)
PyObject* token_scores(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded_call(n, 3, [&]() -> Tensors {
    const at::Tensor z = tensor(a[0]), t = ids(a[1], z);
    const int64_t top = integer(a[2]);
    NEED(z.dim() >= 1 && t.sizes() == z.sizes().slice(0, z.dim() - 1) && real(z.scalar_type()) && (z.is_contiguous() || z.dim() == 2));
    NEED(top >= 0 && top <= FPB_MAX_TOP && top <= z.size(-1) && z.size(-1) <= 1 << 30);
    Scores::stride(z);
    Tensors r = graph_wanted({z}) ? Scores::apply(z, t, top) : Scores::run(z, t, top);
    r.resize(4);
    return r;
  });
}

// address(t, dtype, align, device_index, n0, n1) -> address of a contiguous parameter of that shape (n1 = 0: one dimension), or None
PyObject* address(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, [&]() -> PyObject* {
    const at::Tensor t = tensor(a[0]);
    NEED(THPDtype_Check(a[1]) && t.scalar_type() == reinterpret_cast<THPDtype*>(a[1])->scalar_type && t.device().index() == integer(a[3]));
    const int64_t n0 = integer(a[4]), n1 = integer(a[5]);
    NEED(t.dim() == (n1 ? 2 : 1) && t.size(0) == n0 && (!n1 || t.size(1) == n1) && t.is_contiguous());
    const uintptr_t p = (uintptr_t)t.data_ptr();
    NEED(p % (uintptr_t)integer(a[2]) == 0);
    return PyLong_FromUnsignedLongLong(p);
  });
}

// wanted(ctx) -> per tensor input of the autograd Function whose backward runs, whether this backward uses its gradient:
// an input that requires none, or that autograd.grad(..., inputs) leaves out, does not (needs_input_grad tells the first only)
PyObject* wanted(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 1 || !THPFunction_Check(a[0])) Py_RETURN_NONE;
  const auto node = reinterpret_cast<THPFunction*>(a[0])->cdata.lock();
  if (!node) Py_RETURN_NONE;
  const Py_ssize_t outputs = (Py_ssize_t)node->num_outputs();
  PyObject* r = PyTuple_New(outputs);
  if (!r) return nullptr;
  for (Py_ssize_t i = 0; i < outputs; ++i) PyTuple_SET_ITEM(r, i, PyBool_FromLong(node->task_should_compute_output((size_t)i)));
  return r;
}

// capturable() -> (): raises where the node that runs must not be part of a capture
PyObject* capturable(PyObject*, PyObject* const*, Py_ssize_t n) {
  return guarded_call(n, 0, []() -> Tensors {
    may_be_captured();
    return {};
  });
}

// bind(addresses): the C ABI's entry points in the order of `Entry`
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != ENTRIES) { PyErr_SetString(PyExc_TypeError, "wrong number of entry points"); return nullptr; }
  void* p[ENTRIES];
  for (int i = 0; i < ENTRIES; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null entry point"); return nullptr; }
  }
  memcpy(&entry, p, sizeof(entry));
  Py_RETURN_NONE;
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST(step), FAST(forward), FAST(backward), FAST(suffix_forward), FAST(suffix_backward), FAST(rotary), FAST(gate_forward),
                         FAST(gate_backward), FAST(norm_forward), FAST(norm_backward), FAST(column_sums), FAST(qk_norm_rotary), FAST(dropout),
                         FAST(embedding), FAST(token_scores), FAST(address), FAST(wanted), FAST(capturable), FAST(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "fpb_fast_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_fpb_fast_calls(void) { return PyModule_Create(&module); }
