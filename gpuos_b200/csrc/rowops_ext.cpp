// The row operators (gpuos_rotary, gpuos_cache_*, gpuos_attend, gpuos_route*, gpuos_order, gpuos_dispatch, gpuos_combine*,
// gpuos_logprobs*, gpuos_verify)
// in the Python module `gpuos_ext`: tensors in, new or given tensors out, on
// torch's current stream of the tensors' device.  gpuos_b200/rowops.py is what
// callers use; it adds gradients and the order after a scheduler's requests.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty_like.h>
#include <ATen/TracerMode.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "../../include/gpuos_b200.h"

// rowops.cpp
extern "C" int32_t gpuos_rowops_enter(int32_t device);
extern "C" void gpuos_rowops_leave(int32_t before);

namespace {

// A failed check: raised as the Python exception `type`.
struct Raise {
  PyObject* type;
  std::string msg;
};

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw Raise{PyExc_TypeError, std::string(name) + " must be a torch.Tensor"};
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda())
    throw Raise{PyExc_RuntimeError, "tensors must be CUDA (" + std::string(name) + " is on " + t.device().str() + ")"};
  return t;
}

gpuos_tensor describe(const at::Tensor& t, const char* name) {
  gpuos_tensor d;
  switch (t.scalar_type()) {
    case at::kFloat: d.dtype = GPUOS_F32; break;
    case at::kHalf: d.dtype = GPUOS_F16; break;
    case at::kBFloat16: d.dtype = GPUOS_BF16; break;
    case at::kInt: d.dtype = GPUOS_I32; break;
    case at::kDouble: d.dtype = GPUOS_F64; break;
    case at::kLong: d.dtype = GPUOS_I64; break;
    case at::kByte: d.dtype = GPUOS_U8; break;
    case at::kChar: d.dtype = GPUOS_I8; break;
    case at::kFloat8_e4m3fn: d.dtype = GPUOS_E4M3; break;
    default:
      throw Raise{PyExc_TypeError, std::string(name) + ": dtype " + c10::toString(t.scalar_type()) + " is not supported"};
  }
  if (t.is_conj() || t.is_neg() || t.layout() != at::kStrided)
    throw Raise{PyExc_TypeError, std::string(name) + " must be a plain strided tensor"};
  const int64_t nd = t.dim();
  if (nd > 8) throw Raise{PyExc_ValueError, std::string(name) + " has more than 8 dims"};
  d.ndim = (int32_t)nd;
  d.data = t.numel() ? const_cast<void*>(t.const_data_ptr()) : nullptr;
  for (int64_t i = 0; i < nd; ++i) {
    d.sizes[i] = t.size(i);
    d.strides[i] = t.stride(i);
  }
  return d;
}

// The device of a call's first tensor: made current, with its current stream;
// the other tensors must be on it.
struct Place {
  c10::Device device;
  c10::cuda::CUDAGuard guard;
  int32_t before;
  explicit Place(const at::Tensor& t)
      : device(t.device()), guard(t.device()), before(gpuos_rowops_enter(t.device().index())) {}
  Place(const Place&) = delete;
  ~Place() { gpuos_rowops_leave(before); }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }
  gpuos_tensor in(const at::Tensor& t, const char* name) const {
    if (t.device() != device) throw Raise{PyExc_RuntimeError, "device mismatch"};
    return describe(t, name);
  }
  gpuos_tensor in(PyObject* o, const char* name) const { return in(tensor(o, name), name); }
  // A new contiguous tensor with a storage of its own, as torch.empty's: without the latter's
  // choices, which cost a call of several outputs about as much as all checks.
  at::Tensor make(at::IntArrayRef sizes, at::ScalarType type) const {
    int64_t bytes = (int64_t)c10::elementSize(type);
    for (const int64_t d : sizes)
      if (d < 0 || __builtin_mul_overflow(bytes, d, &bytes)) throw Raise{PyExc_ValueError, "an output is too large"};
    c10::Allocator* const from = c10::cuda::CUDACachingAllocator::get();
    const at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(
        c10::make_intrusive<c10::StorageImpl>(c10::StorageImpl::use_byte_size_t(), (size_t)bytes,
                                              from->allocate((size_t)bytes), from, /*resizable=*/true),
        c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    return t;
  }
};

void done(int32_t rc) {
  if (rc == GPUOS_OK) return;
  const char* msg = gpuos_last_error();
  throw Raise{rc == GPUOS_EINVAL ? PyExc_ValueError : PyExc_RuntimeError, (msg && *msg) ? msg : "gpuos error"};
}

void arity(Py_ssize_t n, Py_ssize_t want, const char* usage) {
  if (n != want) throw Raise{PyExc_TypeError, std::string("expected ") + usage};
}

struct PyFailed {};  // a Python error is set

long integer(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw PyFailed{};
  return v;
}

int32_t small(PyObject* o, const char* name) {
  const long v = integer(o);
  if (v < INT32_MIN || v > INT32_MAX) throw Raise{PyExc_ValueError, std::string(name) + " is out of range"};
  return (int32_t)v;
}

double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PyFailed{};
  return v;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PyFailed{};
  return v != 0;
}

// One tensor, or a tuple of one or two.
struct Pair {
  PyObject* o[2] = {nullptr, nullptr};
  int n = 1;
  bool tuple = false;
  Pair(PyObject* arg, const char* name) {
    if (!PyTuple_Check(arg)) {
      o[0] = arg;
      return;
    }
    tuple = true;
    n = (int)PyTuple_GET_SIZE(arg);
    if (n < 1 || n > 2)
      throw Raise{PyExc_TypeError, std::string(name) + " must be a tensor, or a tuple of one or two tensors"};
    for (int i = 0; i < n; ++i) o[i] = PyTuple_GET_ITEM(arg, i);
  }
};

PyObject* wrap(const at::Tensor& t) {
  PyObject* o = THPVariable_Wrap(t);
  if (!o) throw PyFailed{};
  return o;
}

// Whether torch has to see the call (gpuos_b200.rowops then makes it an autograd function's): for
// a gradient, or for a tangent of forward mode.
bool recorded(const at::Tensor& t) {
  const c10::AutogradState& state = c10::AutogradState::get_tls_state();
  return (state.get_grad_mode() && t.requires_grad()) || (state.get_fw_grad_mode() && t._fw_grad(0).defined());
}

// A call whose result torch.jit.trace would take for a constant: to be made an autograd function's, which
// is an operation of the trace, or refused.  Inside such a function forward mode is off; in
// inference mode it is off everywhere, so that nothing tells the two apart.
bool tracing() { return at::tracer::impl::is_dispatch_enabled(); }
void not_traced() {
  if (tracing()) throw Raise{PyExc_RuntimeError, "torch.jit.trace cannot record this call"};
}
bool traced() {
  if (!tracing()) return false;
  if (c10::AutogradState::get_tls_state().get_inference_mode()) not_traced();
  return c10::AutogradState::get_tls_state().get_fw_grad_mode();
}

// A tensor of the caller's was written: autograd then refuses a backward pass that saved it.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A tensor to be written, which autograd must not be following.
const at::Tensor& given_out(PyObject* o, const char* name = "out") {
  const at::Tensor& t = tensor(o, name);
  if (recorded(t)) throw Raise{PyExc_ValueError, std::string(name) + " cannot be a tensor that requires a gradient"};
  return t;
}

PyObject* not_here() {
  Py_INCREF(Py_NotImplemented);
  return Py_NotImplemented;
}

void same_count(Py_ssize_t a, Py_ssize_t b, const char* what) {
  if (a != b) throw Raise{PyExc_ValueError, what};
}

PyObject* tuple_of(const at::Tensor* t, Py_ssize_t n) {
  PyObject* r = PyTuple_New(n);
  if (!r) throw PyFailed{};
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o;
    if (t[i].defined()) {
      o = THPVariable_Wrap(t[i]);
    } else {
      o = Py_None;
      Py_INCREF(o);
    }
    if (!o) {
      Py_DECREF(r);
      throw PyFailed{};
    }
    PyTuple_SET_ITEM(r, i, o);
  }
  return r;
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  try {
    return F(args, n);
  } catch (const Raise& r) {
    PyErr_SetString(r.type, r.msg.c_str());
    return nullptr;
  } catch (const PyFailed&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

PyObject* rotary(PyObject* const* a, Py_ssize_t n) {
  arity(n, 7, "(x, out, positions, inv_freq, scale, interleaved, inverse)");
  const Pair xs(a[0], "x");
  const at::Tensor* xt[2];
  if (recorded(tensor(a[3], "inv_freq")))
    throw Raise{PyExc_ValueError, "inv_freq takes no gradient: detach it"};
  for (int i = 0; i < xs.n; ++i) {
    xt[i] = &tensor(xs.o[i], "x");
    if (recorded(*xt[i]) || traced()) return not_here();
  }
  const Place at(*xt[0]);
  gpuos_tensor x[2], o[2];
  at::Tensor out[2];
  if (a[1] != Py_None) {
    const Pair given(a[1], "out");
    same_count(given.n, xs.n, "out must have a tensor for each x");
    for (int i = 0; i < xs.n; ++i) out[i] = given_out(given.o[i]);
  } else {
    for (int i = 0; i < xs.n; ++i) {
      // the layout of x, where its last dim is contiguous in it
      const bool plain = xt[i]->is_contiguous();
      if (!plain) out[i] = at::empty_like(*xt[i]);
      if (plain || (xt[i]->dim() && out[i].stride(-1) != 1)) out[i] = at.make(xt[i]->sizes(), xt[i]->scalar_type());
    }
  }
  for (int i = 0; i < xs.n; ++i) {
    x[i] = at.in(*xt[i], "x");
    o[i] = at.in(out[i], "out");
  }
  const gpuos_tensor p = at.in(a[2], "positions"), f = at.in(a[3], "inv_freq");
  const double scale = real(a[4]);
  const int32_t flags = (truth(a[5]) ? GPUOS_ROTARY_INTERLEAVED : 0) | (truth(a[6]) ? GPUOS_ROTARY_INVERSE : 0);
  done(gpuos_rotary(xs.n, x, o, &p, &f, (float)scale, flags, at.stream()));
  if (a[1] != Py_None)
    for (int i = 0; i < xs.n; ++i) written(out[i]);
  return xs.tuple ? tuple_of(out, xs.n) : wrap(out[0]);
}

PyObject* cache_write(PyObject* const* a, Py_ssize_t n) {
  arity(n, 4, "(x, slots, codes, scales)");
  not_traced();
  const Pair xs(a[0], "x"), cs(a[2], "codes"), ss(a[3], "scales");
  same_count(cs.n, xs.n, "codes must have a tensor for each x");
  same_count(ss.n, xs.n, "scales must have a tensor for each x");
  const Place at(tensor(xs.o[0], "x"));
  gpuos_tensor x[2], c[2], s[2];
  for (int i = 0; i < xs.n; ++i) {
    x[i] = at.in(xs.o[i], "x");
    c[i] = at.in(given_out(cs.o[i], "codes"), "codes");
    s[i] = at.in(given_out(ss.o[i], "scales"), "scales");
  }
  const gpuos_tensor slots = at.in(a[1], "slots");
  done(gpuos_cache_write(xs.n, x, &slots, c, s, at.stream()));
  for (int i = 0; i < xs.n; ++i) {
    written(tensor(cs.o[i], "codes"));
    written(tensor(ss.o[i], "scales"));
  }
  Py_RETURN_NONE;
}

PyObject* cache_read(PyObject* const* a, Py_ssize_t n) {
  arity(n, 5, "(slots, codes, scales, out, dtype)");
  not_traced();
  const Pair cs(a[1], "codes"), ss(a[2], "scales");
  same_count(ss.n, cs.n, "scales must have a tensor for each cache");
  const at::Tensor& slots_t = tensor(a[0], "slots");
  const Place at(slots_t);
  gpuos_tensor c[2], s[2], o[2];
  at::Tensor out[2];
  if (a[3] != Py_None) {
    const Pair given(a[3], "out");
    same_count(given.n, cs.n, "out must have a tensor for each cache");
    for (int i = 0; i < cs.n; ++i) out[i] = given_out(given.o[i]);
  }
  const int32_t code = small(a[4], "dtype");
  const at::ScalarType type = code == GPUOS_F32 ? at::kFloat : code == GPUOS_F16 ? at::kHalf : at::kBFloat16;
  for (int i = 0; i < cs.n; ++i) {
    const at::Tensor& codes = tensor(cs.o[i], "codes");
    c[i] = at.in(codes, "codes");
    s[i] = at.in(ss.o[i], "scales");
    if (a[3] != Py_None) continue;
    if (codes.dim() != 4 || slots_t.dim() != 1)
      throw Raise{PyExc_ValueError, "codes must be (page, row, head, code) and slots have one dim"};
    out[i] = at.make({slots_t.size(0), codes.size(2), codes.size(3) * (codes.scalar_type() == at::kByte ? 2 : 1)}, type);
  }
  for (int i = 0; i < cs.n; ++i) o[i] = at.in(out[i], "out");
  const gpuos_tensor slots = at.in(slots_t, "slots");
  done(gpuos_cache_read(cs.n, &slots, c, s, o, at.stream()));
  if (a[3] != Py_None)
    for (int i = 0; i < cs.n; ++i) written(out[i]);
  return cs.tuple ? tuple_of(out, cs.n) : wrap(out[0]);
}

PyObject* attend(PyObject* const* a, Py_ssize_t n) {
  arity(n, 12, "(q, codes, scales, pages, lengths, offsets, longest, causal, window, scale, lse, out)");
  not_traced();
  const at::Tensor& x = tensor(a[0], "q");
  if (recorded(x)) throw Raise{PyExc_ValueError, "q takes no gradient here: detach it"};
  const Pair cs(a[1], "codes"), ss(a[2], "scales");
  if (cs.n != 2 || ss.n != 2) throw Raise{PyExc_ValueError, "codes and scales must have a tensor each for keys and for values"};
  const Place at(x);
  const gpuos_tensor q = at.in(x, "q");
  gpuos_tensor c[2], s[2], offsets;
  for (int i = 0; i < 2; ++i) {
    c[i] = at.in(cs.o[i], "codes");
    s[i] = at.in(ss.o[i], "scales");
  }
  const gpuos_tensor pages = at.in(a[3], "pages"), lengths = at.in(a[4], "lengths");
  const bool ragged = a[5] != Py_None;
  if (ragged) offsets = at.in(a[5], "offsets");
  if (x.dim() != 3) throw Raise{PyExc_ValueError, "q must have 3 dims, not " + std::to_string(x.dim())};
  const int64_t longest = a[6] != Py_None ? (int64_t)integer(a[6]) : ragged ? std::max<int64_t>(x.size(0), 1) : 1;
  const int64_t window = a[8] != Py_None ? (int64_t)integer(a[8]) : 0;
  if (a[8] != Py_None && window < 1) throw Raise{PyExc_ValueError, "window must be at least 1"};
  const double scale = a[9] != Py_None ? real(a[9]) : 1.0 / std::sqrt((double)std::max<int64_t>(x.size(2), 1));
  const at::Tensor out = a[11] != Py_None ? given_out(a[11]) : at.make(x.sizes(), x.scalar_type());
  const gpuos_tensor o = at.in(out, "out");
  at::Tensor lse, work;
  gpuos_tensor l;
  if (truth(a[10])) {
    lse = at.make({x.size(0), x.size(1)}, at::kFloat);
    l = at.in(lse, "lse");
  }
  int64_t bytes = 0;
  done(gpuos_attend_workspace(&q, &c[0], &s[0], &pages, longest, &bytes));
  if (bytes) work = at.make({bytes}, at::kByte);
  done(gpuos_attend(&q, c, s, &pages, &lengths, ragged ? &offsets : nullptr, &o, lse.defined() ? &l : nullptr,
                    bytes ? const_cast<void*>(work.const_data_ptr()) : nullptr, bytes, longest, window, (float)scale,
                    truth(a[7]) ? GPUOS_ATTEND_CAUSAL : 0, at.stream()));
  if (a[11] != Py_None) written(out);
  if (!lse.defined()) return wrap(out);
  const at::Tensor both[2] = {out, lse};
  return tuple_of(both, 2);
}

PyObject* route(PyObject* const* a, Py_ssize_t n) {
  arity(n, 9, "(logits, bias, top_k, score, groups, top_groups, group_score, renormalize, scale)");
  const at::Tensor& x = tensor(a[0], "logits");
  if (recorded(x) || traced()) return not_here();
  const Place at(x);
  const gpuos_tensor d = at.in(x, "logits");
  if (x.dim() != 2) throw Raise{PyExc_ValueError, "logits must have 2 dims, not " + std::to_string(x.dim())};
  gpuos_tensor bias;
  if (a[1] != Py_None) bias = at.in(a[1], "bias");
  const int32_t k = small(a[2], "top_k");
  if (k < 1 || k > 64) throw Raise{PyExc_ValueError, "top_k must be in [1, 64]"};
  const at::Tensor out[2] = {at.make({x.size(0), k}, at::kFloat), at.make({x.size(0), k}, at::kLong)};
  const gpuos_tensor w = at.in(out[0], "weights"), e = at.in(out[1], "experts");
  done(gpuos_route(&d, a[1] != Py_None ? &bias : nullptr, &w, &e, small(a[3], "score"), small(a[4], "groups"),
                   small(a[5], "top_groups"), small(a[6], "group_score"), truth(a[7]), (float)real(a[8]), at.stream()));
  return tuple_of(out, 2);
}

PyObject* route_grad(PyObject* const* a, Py_ssize_t n) {
  arity(n, 6, "(logits, experts, grad_weights, score, renormalize, scale)");
  not_traced();
  const at::Tensor& x = tensor(a[0], "logits");
  const Place at(x);
  const gpuos_tensor d = at.in(x, "logits"), e = at.in(a[1], "experts"), g = at.in(a[2], "grad_weights");
  const at::Tensor out = at.make(x.sizes(), x.scalar_type());
  const gpuos_tensor o = at.in(out, "grad_logits");
  done(gpuos_route_grad(&d, &e, &g, &o, small(a[3], "score"), truth(a[4]), (float)real(a[5]), at.stream()));
  return wrap(out);
}

PyObject* logprobs(PyObject* const* a, Py_ssize_t n) {
  arity(n, 6, "(logits, targets, top, entropy, temperature, stats)");
  const at::Tensor& x = tensor(a[0], "logits");
  if (recorded(x) || traced()) return not_here();
  const Place at(x);
  const gpuos_tensor d = at.in(x, "logits"), y = at.in(a[1], "targets");
  if (x.dim() != 2) throw Raise{PyExc_ValueError, "logits must have 2 dims, not " + std::to_string(x.dim())};
  const int32_t k = small(a[2], "top");
  if (k < 0 || k > 64) throw Raise{PyExc_ValueError, "top must be in [0, 64]"};
  const bool entropy = truth(a[3]), stats = truth(a[5]);
  const int64_t rows = x.size(0);
  at::Tensor out[5];  // logprob, entropy, top_logprobs, top_tokens, stats
  out[0] = at.make({rows}, at::kFloat);
  if (entropy) out[1] = at.make({rows}, at::kFloat);
  if (k) {
    out[2] = at.make({rows, k}, at::kFloat);
    out[3] = at.make({rows, k}, at::kLong);
  }
  if (stats) out[4] = at.make({rows, 2}, at::kFloat);
  gpuos_tensor o[5];
  for (int i = 0; i < 5; ++i)
    if (out[i].defined()) o[i] = at.in(out[i], "out");
  done(gpuos_logprobs(&d, &y, &o[0], entropy ? &o[1] : nullptr, k ? &o[2] : nullptr, k ? &o[3] : nullptr,
                      stats ? &o[4] : nullptr, (float)real(a[4]), at.stream()));
  return tuple_of(out, 5);
}

PyObject* logprobs_grad(PyObject* const* a, Py_ssize_t n) {
  arity(n, 8, "(logits, targets, stats, entropy, grad_logprob, grad_entropy, temperature, out)");
  not_traced();
  const at::Tensor& x = tensor(a[0], "logits");
  const Place at(x);
  const gpuos_tensor d = at.in(x, "logits"), y = at.in(a[1], "targets"), st = at.in(a[2], "stats");
  gpuos_tensor opt[3];
  const char* names[3] = {"entropy", "grad_logprob", "grad_entropy"};
  for (int i = 0; i < 3; ++i)
    if (a[3 + i] != Py_None) opt[i] = at.in(a[3 + i], names[i]);
  const at::Tensor out = a[7] != Py_None ? given_out(a[7]) : at.make(x.sizes(), x.scalar_type());
  const gpuos_tensor o = at.in(out, "out");
  done(gpuos_logprobs_grad(&d, &y, &st, a[3] != Py_None ? &opt[0] : nullptr, a[4] != Py_None ? &opt[1] : nullptr,
                           a[5] != Py_None ? &opt[2] : nullptr, &o, (float)real(a[6]), at.stream()));
  if (a[7] != Py_None) written(out);
  return wrap(out);
}

// The order of a token's choices: (places, sources, ...) as a tuple.
struct Given {
  const at::Tensor *places, *sources;
  gpuos_tensor p, s;
  Given(const Place& at, PyObject* o) {
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 4) throw Raise{PyExc_TypeError, "order must be what rowops.order returned"};
    places = &tensor(PyTuple_GET_ITEM(o, 0), "places");
    sources = &tensor(PyTuple_GET_ITEM(o, 1), "sources");
    p = at.in(*places, "places");
    s = at.in(*sources, "sources");
    if (places->dim() != 2 || sources->dim() != 1)
      throw Raise{PyExc_ValueError, "order: places must be (token, choice) and sources have one dim"};
  }
};

void two_dims(const at::Tensor& t, const char* name) {
  if (t.dim() != 2) throw Raise{PyExc_ValueError, std::string(name) + " must have 2 dims, not " + std::to_string(t.dim())};
}

PyObject* order(PyObject* const* a, Py_ssize_t n) {
  arity(n, 3, "(experts, count, align)");
  not_traced();
  const at::Tensor& x = tensor(a[0], "experts");
  const Place at(x);
  const gpuos_tensor d = at.in(x, "experts");
  two_dims(x, "experts");
  const int32_t count = small(a[1], "count"), align = small(a[2], "align");
  if (count < 1 || count > 1024) throw Raise{PyExc_ValueError, "count must be in [1, 1024]"};
  int64_t rows = 0;
  done(gpuos_order_rows(x.numel(), count, align, &rows));
  const at::Tensor out[4] = {at.make(x.sizes(), at::kInt), at.make({rows}, at::kInt), at.make({count + 1}, at::kInt),
                             at.make({count}, at::kInt)};
  const gpuos_tensor o[4] = {at.in(out[0], "places"), at.in(out[1], "sources"), at.in(out[2], "offsets"), at.in(out[3], "counts")};
  done(gpuos_order(&d, align, &o[0], &o[1], &o[2], &o[3], at.stream()));
  return tuple_of(out, 4);
}

PyObject* dispatch(PyObject* const* a, Py_ssize_t n) {
  arity(n, 2, "(x, order)");
  const at::Tensor& x = tensor(a[0], "x");
  if (recorded(x) || traced()) return not_here();
  const Place at(x);
  const Given by(at, a[1]);
  const gpuos_tensor d = at.in(x, "x");
  two_dims(x, "x");
  const at::Tensor out = at.make({by.sources->size(0), x.size(1)}, x.scalar_type());
  const gpuos_tensor o = at.in(out, "rows");
  done(gpuos_dispatch(&d, &by.p, &by.s, &o, at.stream()));
  return wrap(out);
}

PyObject* combine(PyObject* const* a, Py_ssize_t n) {
  arity(n, 3, "(y, order, weights)");
  const at::Tensor& y = tensor(a[0], "y");
  if (recorded(y) || traced() || (a[2] != Py_None && recorded(tensor(a[2], "weights")))) return not_here();
  const Place at(y);
  const Given by(at, a[1]);
  const gpuos_tensor d = at.in(y, "y");
  two_dims(y, "y");
  gpuos_tensor w;
  if (a[2] != Py_None) w = at.in(a[2], "weights");
  const at::Tensor out = at.make({by.places->size(0), y.size(1)}, y.scalar_type());
  const gpuos_tensor o = at.in(out, "out");
  done(gpuos_combine(&d, &by.p, &by.s, a[2] != Py_None ? &w : nullptr, &o, at.stream()));
  return wrap(out);
}

PyObject* combine_grad(PyObject* const* a, Py_ssize_t n) {
  arity(n, 6, "(grad, y, order, weights, want_y, want_weights)");
  not_traced();
  const at::Tensor& g = tensor(a[0], "grad");
  const Place at(g);
  const Given by(at, a[2]);
  const gpuos_tensor d = at.in(g, "grad"), w = at.in(a[3], "weights");
  two_dims(g, "grad");
  const bool want[2] = {truth(a[4]), truth(a[5])};
  gpuos_tensor y, o[2];
  if (a[1] != Py_None) y = at.in(a[1], "y");
  at::Tensor out[2];
  if (want[0]) out[0] = at.make({by.sources->size(0), g.size(1)}, g.scalar_type());
  if (want[1]) out[1] = at.make(by.places->sizes(), at::kFloat);
  for (int i = 0; i < 2; ++i)
    if (want[i]) o[i] = at.in(out[i], i ? "grad_weights" : "grad_y");
  done(gpuos_combine_grad(&d, a[1] != Py_None ? &y : nullptr, &by.p, &by.s, &w, want[0] ? &o[0] : nullptr,
                          want[1] ? &o[1] : nullptr, at.stream()));
  return tuple_of(out, 2);
}

PyObject* verify(PyObject* const* a, Py_ssize_t n) {
  arity(n, 5, "(logits, drafts, uniforms, probs, temperature)");
  not_traced();
  const at::Tensor& x = tensor(a[0], "logits");
  const Place at(x);
  const gpuos_tensor d = at.in(x, "logits"), y = at.in(a[1], "drafts");
  if (x.dim() != 3) throw Raise{PyExc_ValueError, "logits must have 3 dims, not " + std::to_string(x.dim())};
  gpuos_tensor u, q;
  if (a[2] != Py_None) u = at.in(a[2], "uniforms");
  if (a[3] != Py_None) q = at.in(a[3], "probs");
  const at::Tensor out[2] = {at.make({x.size(0), x.size(1)}, at::kLong), at.make({x.size(0)}, at::kLong)};
  const gpuos_tensor o[2] = {at.in(out[0], "tokens"), at.in(out[1], "accepted")};
  done(gpuos_verify(&d, &y, a[2] != Py_None ? &u : nullptr, a[3] != Py_None ? &q : nullptr, &o[0], &o[1], real(a[4]),
                    at.stream()));
  return tuple_of(out, 2);
}

}  // namespace

#define GPUOS_FAST(f) (PyCFunction)(void (*)(void))guarded<f>, METH_FASTCALL

PyMethodDef* gpuos_rowops_methods() {
  static PyMethodDef methods[] = {
      {"rotary", GPUOS_FAST(rotary), "rotary(x, out, positions, inv_freq, scale, interleaved, inverse): see rowops.rotary"},
      {"cache_write", GPUOS_FAST(cache_write), "cache_write(x, slots, codes, scales): see rowops.cache_write"},
      {"cache_read", GPUOS_FAST(cache_read), "cache_read(slots, codes, scales, out, dtype): see rowops.cache_read"},
      {"attend", GPUOS_FAST(attend),
       "attend(q, codes, scales, pages, lengths, offsets, longest, causal, window, scale, lse, out): see rowops.attend"},
      {"route", GPUOS_FAST(route),
       "route(logits, bias, top_k, score, groups, top_groups, group_score, renormalize, scale): see rowops.route"},
      {"route_grad", GPUOS_FAST(route_grad),
       "route_grad(logits, experts, grad_weights, score, renormalize, scale): see rowops.route_grad"},
      {"logprobs", GPUOS_FAST(logprobs), "logprobs(logits, targets, top, entropy, temperature, stats): see rowops.logprobs"},
      {"logprobs_grad", GPUOS_FAST(logprobs_grad),
       "logprobs_grad(logits, targets, stats, entropy, grad_logprob, grad_entropy, temperature, out): see "
       "rowops.logprobs_grad"},
      {"order", GPUOS_FAST(order), "order(experts, count, align): see rowops.order"},
      {"dispatch", GPUOS_FAST(dispatch), "dispatch(x, order): see rowops.dispatch"},
      {"combine", GPUOS_FAST(combine), "combine(y, order, weights): see rowops.combine"},
      {"combine_grad", GPUOS_FAST(combine_grad),
       "combine_grad(grad, y, order, weights, want_y, want_weights): see rowops.combine_grad"},
      {"verify", GPUOS_FAST(verify), "verify(logits, drafts, uniforms, probs, temperature): see rowops.verify"},
      {nullptr, nullptr, 0, nullptr}};
  return methods;
}
