// The short way from a torch call to the sequence-policy operators (_calls, a CPython module over torch's C++ API).
//
// A call through ctypes costs 10 to 25 us on the host, most of it spent in Python's attribute lookups, argument
// conversions and allocations; that is more than these operators take on the GPU for the sizes that
// generation and small updates call them with.  Here the same checks, allocations and the call of the C ABI
// (include/b200ops.h) are done in C++.  Each function takes the ordinary case of the operator it is named
// after; for anything else (a wrong argument, an empty tensor, another device than the current one, a call that is
// being captured into a graph and needs scratch) it returns None, and the caller in ops.py goes its own way, which
// also says what is wrong.
//
// Scratch is kept per operator, device and stream, zero-filled when it is made, apart from the scratch of ops.py.
// The caller holds ops.py's launch lock: a call may be two launches, which those of another thread must not part.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <cstring>
#include <map>
#include <optional>
#include <tuple>

#include "../../../include/b200ops.h"

namespace {

using at::Tensor;
constexpr int64_t kMax = 0x7fffffff;

PyObject* g_error = nullptr;  // OpError

// The entry points, found by name in the library that init() is given.
#define ENTRY(name) decltype(&::name) name##_ = nullptr
ENTRY(b200_status_string);
ENTRY(b200_linear_recurrence_checkpoint_bytes);
ENTRY(b200_linear_recurrence_workspace_bytes);
ENTRY(b200_linear_recurrence_async);
ENTRY(b200_linear_recurrence_backward_async);
ENTRY(b200_linear_recurrence_step_async);
ENTRY(b200_token_logprob_async);
ENTRY(b200_token_logprob_backward_async);
ENTRY(b200_policy_loss_workspace_bytes);
ENTRY(b200_policy_loss_async);
ENTRY(b200_preference_loss_workspace_bytes);
ENTRY(b200_preference_loss_async);

// Other threads run Python while a call allocates and launches (a launch waits when the GPU's queue is full).
template <typename F>
int unlocked(F&& f) {
  struct NoGil {
    PyThreadState* state = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(state); }
  } no_gil;
  return f();
}

// What a call works on: the current device and its current stream.
struct Place {
  c10::Device device;
  cudaStream_t stream;
};

// A plain torch tensor (or parameter) argument; null otherwise.
const Tensor* tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const Tensor* t = &THPVariable_Unpack(o);
  return t->layout() == at::kStrided && !t->is_nested() ? t : nullptr;
}

// The number of a form, -1 for anything else.
int form_of(PyObject* o) {
  if (!PyLong_CheckExact(o)) return -1;
  int overflow;
  const long v = PyLong_AsLongAndOverflow(o, &overflow);
  return overflow == 0 && v >= 0 && v < 16 ? int(v) : -1;
}

// None or a tensor: false when it is neither.
bool optional_tensor(PyObject* o, const Tensor** t) {
  *t = nullptr;
  if (o == Py_None) return true;
  *t = tensor(o);
  return *t != nullptr;
}

bool place_of(const Tensor& t, std::optional<Place>* p) {
  if (!t.is_cuda() || t.device().index() != c10::cuda::current_device()) return false;
  *p = Place{t.device(), at::cuda::getCurrentCUDAStream(t.device().index()).stream()};
  return true;
}

// dtype codes of the C ABI (-1: another type).
int code_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return B200_F32;
    case at::kBFloat16: return B200_BF16;
    case at::kHalf: return B200_F16;
    default: return -1;
  }
}

// Elements that the last axis holds one behind another, of the given type, on the call's device.
bool rows(const Tensor& t, const Place& p, at::ScalarType type, int64_t dims) {
  return t.dim() == dims && t.scalar_type() == type && t.device() == p.device && t.numel() > 0 && t.numel() <= 64 * kMax &&
         (t.stride(-1) == 1 || t.size(-1) == 1);
}
bool dense(const Tensor& t, const Place& p, at::ScalarType type, at::IntArrayRef shape) {
  return t.scalar_type() == type && t.device() == p.device && t.sizes() == shape && t.is_contiguous();
}
// An optional [B, T] stream with contiguous tokens.
bool stream_ok(const Tensor* t, const Place& p, at::ScalarType type, int64_t B, int64_t T) {
  return t == nullptr || (rows(*t, p, type, 2) && t->size(0) == B && t->size(1) == T);
}
int64_t row_stride(const Tensor* t) { return t == nullptr ? 0 : t->stride(0); }
void* at_(const Tensor* t) { return t == nullptr || !t->defined() ? nullptr : t->data_ptr(); }
template <typename T>
T* ptr(const Tensor* t) {
  return static_cast<T*>(at_(t));
}

// Whether two tensors span different memory.
bool apart(const Tensor& a, const Tensor& b) {
  const auto last = [](const Tensor& t) {
    int64_t n = 1;
    for (int64_t d = 0; d < t.dim(); ++d) n += (t.size(d) - 1) * t.stride(d);
    return static_cast<const char*>(t.data_ptr()) + n * int64_t(t.element_size());
  };
  return last(a) <= static_cast<const char*>(b.data_ptr()) || last(b) <= static_cast<const char*>(a.data_ptr());
}

// A new tensor, without the way through torch's dispatcher.
Tensor make(at::IntArrayRef shape, at::ScalarType type, const Place& p) {
  return at::detail::empty_cuda(shape, type, p.device, std::nullopt);
}

enum Op { kRecurrence, kPolicy, kPreference };

// The scratch of an operator on the call's stream (never freed: the driver may be gone before static objects are).
// null while the stream is being captured.
const Tensor* scratch(Op op, int64_t bytes, const Place& p) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return nullptr;
  static auto* all = new std::map<std::tuple<int, int, cudaStream_t>, Tensor>();
  Tensor& t = (*all)[{int(op), int(p.device.index()), p.stream}];
  if (!t.defined() || t.numel() < bytes)
    t = at::zeros({bytes < 4096 ? 4096 : bytes}, at::TensorOptions().dtype(at::kByte).device(p.device));
  return &t;
}

// Outputs on success, an exception otherwise.
PyObject* wrap(const Tensor* t) {
  if (t == nullptr || !t->defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(*t);
}
template <typename... Ts>
PyObject* done(int status, const char* what, const Ts&... t) {
  if (status != 0) {
    PyErr_Format(g_error, "%s: status %d (%s)", what, status, b200_status_string_(status));
    return nullptr;
  }
  PyObject* items[] = {wrap(&t)...};
  constexpr Py_ssize_t n = sizeof...(Ts);
  PyObject* tuple = PyTuple_New(n);
  if (tuple == nullptr) {
    for (PyObject* item : items) Py_XDECREF(item);
    return nullptr;
  }
  for (Py_ssize_t i = 0; i < n; ++i) PyTuple_SET_ITEM(tuple, i, items[i]);
  return tuple;
}

#define ORDINARY(condition) \
  do {                      \
    if (!(condition)) Py_RETURN_NONE; \
  } while (0)
// torch's exceptions (out of memory among them) leave as Python's.
#define BEGIN try {
#define END                                              \
  }                                                      \
  catch (const c10::Error& e) {                          \
    PyErr_SetString(c10_error_type(e), e.what_without_backtrace()); \
    return nullptr;                                      \
  }                                                      \
  catch (const std::exception& e) {                      \
    PyErr_SetString(PyExc_RuntimeError, e.what());       \
    return nullptr;                                      \
  }

PyObject* c10_error_type(const c10::Error& e) {
  if (dynamic_cast<const c10::OutOfMemoryError*>(&e) != nullptr) {
    static PyObject* oom = [] {
      PyObject* m = PyImport_ImportModule("torch");
      return m != nullptr ? PyObject_GetAttrString(m, "OutOfMemoryError") : nullptr;
    }();
    if (oom != nullptr) return oom;
    PyErr_Clear();
  }
  return PyExc_RuntimeError;
}

// ------------------------------------------------------------------------ gated linear recurrence
// An output of x's shape and type: dense, time first in memory when x is.
Tensor like_bth(const Tensor& x, const Place& p) {
  const int64_t B = x.size(0), T = x.size(1), H = x.size(2);
  if (B > 1 && T > 1 && x.stride(0) < x.stride(1)) return make({T, B, H}, x.scalar_type(), p).transpose(0, 1);
  return make({B, T, H}, x.scalar_type(), p);
}
bool bth(const Tensor& t, const Tensor& x, const Place& p) {
  return rows(t, p, x.scalar_type(), 3) && t.sizes() == x.sizes();
}
bool state_ok(const Tensor* t, const Place& p, int64_t B, int64_t H) {
  return t == nullptr || dense(*t, p, at::kFloat, {B, H});
}
bool reset_ok(const Tensor* t, const Place& p, int64_t B, int64_t T) {
  return t == nullptr || (t->scalar_type() == at::kBool && t->device() == p.device && t->dim() == 2 && t->size(0) == B &&
                          t->size(1) == T);
}

// recurrence(gate, x, state, reset, form, train) -> (h, final state, checkpoints or None)
PyObject* recurrence(PyObject*, PyObject* const* a, Py_ssize_t n) {
  BEGIN
  const Tensor *gate, *x, *state, *reset;
  ORDINARY(n == 6 && (gate = tensor(a[0])) && (x = tensor(a[1])) && optional_tensor(a[2], &state) &&
           optional_tensor(a[3], &reset));
  std::optional<Place> p;
  const int dtype = code_of(*x), form = form_of(a[4]);
  ORDINARY(dtype >= 0 && form >= 0 && place_of(*x, &p) && bth(*x, *x, *p) && bth(*gate, *x, *p));
  const int64_t B = x->size(0), T = x->size(1), H = x->size(2);
  ORDINARY(B <= kMax && T <= kMax && H <= kMax && state_ok(state, *p, B, H) && reset_ok(reset, *p, B, T));
  const int64_t bytes = b200_linear_recurrence_workspace_bytes_(int(B), int(T), int(H));
  const Tensor* ws = nullptr;
  ORDINARY(bytes == 0 || (ws = scratch(kRecurrence, bytes, *p)) != nullptr);
  Tensor h, final_state, ckpt;
  const bool train = a[5] == Py_True;
  const int status = unlocked([&] {
    h = like_bth(*x, *p), final_state = make({B, H}, at::kFloat, *p);
    if (train) ckpt = make({b200_linear_recurrence_checkpoint_bytes_(int(B), int(T), int(H)) / 4}, at::kFloat, *p);
    const int64_t st[8] = {gate->stride(0), gate->stride(1), x->stride(0), x->stride(1), h.stride(0), h.stride(1),
                           reset ? reset->stride(0) : 0, reset ? reset->stride(1) : 0};
    return b200_linear_recurrence_async_(
        gate->data_ptr(), x->data_ptr(), dtype, form, st, ptr<float>(state), ptr<uint8_t>(reset), int(B), int(T), int(H),
        h.data_ptr(), ptr<float>(&final_state), ptr<float>(&ckpt), at_(ws), ws ? ws->numel() : 0, p->stream);
  });
  return done(status, "linear_recurrence", h, final_state, ckpt);
  END
}

// recurrence_backward(gate, x, checkpoints, grad_h, grad_final, reset, form) -> (grad_gate, grad_x, grad_state)
PyObject* recurrence_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  BEGIN
  const Tensor *gate, *x, *ckpt, *dh, *df, *reset;
  ORDINARY(n == 7 && (gate = tensor(a[0])) && (x = tensor(a[1])) && (ckpt = tensor(a[2])) && (dh = tensor(a[3])) &&
           optional_tensor(a[4], &df) && optional_tensor(a[5], &reset));
  std::optional<Place> p;
  const int dtype = code_of(*x), form = form_of(a[6]);
  ORDINARY(dtype >= 0 && form >= 0 && place_of(*x, &p) && bth(*x, *x, *p) && bth(*gate, *x, *p) && bth(*dh, *x, *p));
  const int64_t B = x->size(0), T = x->size(1), H = x->size(2);
  ORDINARY(B <= kMax && T <= kMax && H <= kMax && state_ok(df, *p, B, H) && reset_ok(reset, *p, B, T));
  ORDINARY(ckpt->scalar_type() == at::kFloat && ckpt->device() == p->device && ckpt->is_contiguous() &&
           ckpt->numel() * 4 == b200_linear_recurrence_checkpoint_bytes_(int(B), int(T), int(H)));
  const int64_t bytes = b200_linear_recurrence_workspace_bytes_(int(B), int(T), int(H));
  const Tensor* ws = nullptr;
  ORDINARY(bytes == 0 || (ws = scratch(kRecurrence, bytes, *p)) != nullptr);
  Tensor gg, gx, gs;
  const int status = unlocked([&] {
    gg = like_bth(*gate, *p), gx = like_bth(*x, *p), gs = make({B, H}, at::kFloat, *p);
    const int64_t st[12] = {gate->stride(0), gate->stride(1), x->stride(0), x->stride(1),
                            dh->stride(0),   dh->stride(1),   gg.stride(0), gg.stride(1),
                            gx.stride(0),    gx.stride(1),    reset ? reset->stride(0) : 0,
                            reset ? reset->stride(1) : 0};
    return b200_linear_recurrence_backward_async_(
        gate->data_ptr(), x->data_ptr(), dtype, form, st, ptr<float>(ckpt), ptr<uint8_t>(reset), dh->data_ptr(),
        ptr<float>(df), int(B), int(T), int(H), gg.data_ptr(), gx.data_ptr(), ptr<float>(&gs), at_(ws),
        ws ? ws->numel() : 0, p->stream);
  });
  return done(status, "linear_recurrence_backward", gg, gx, gs);
  END
}

// recurrence_step(gate, x, state, slots, form, state_out) -> (h,)
PyObject* recurrence_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  BEGIN
  const Tensor *gate, *x, *state, *slots, *next;
  ORDINARY(n == 6 && (gate = tensor(a[0])) && (x = tensor(a[1])) && (state = tensor(a[2])) &&
           optional_tensor(a[3], &slots) && optional_tensor(a[5], &next));
  std::optional<Place> p;
  const int dtype = code_of(*x), form = form_of(a[4]);
  ORDINARY(dtype >= 0 && form >= 0 && place_of(*x, &p) && rows(*x, *p, x->scalar_type(), 2) &&
           rows(*gate, *p, x->scalar_type(), 2) && gate->sizes() == x->sizes());
  const int64_t B = x->size(0), H = x->size(1);
  ORDINARY(B <= kMax && H <= kMax && state->dim() == 2 && state->size(0) <= kMax &&
           dense(*state, *p, at::kFloat, {state->size(0), H}));
  const int64_t S = state->size(0);
  ORDINARY(slots ? dense(*slots, *p, at::kInt, {B}) : S >= B);
  ORDINARY(next == nullptr || (dense(*next, *p, at::kFloat, {S, H}) &&
                               (at_(next) == at_(state) || apart(*next, *state))));
  const Tensor& written = next ? *next : *state;
  ORDINARY(apart(written, *gate) && apart(written, *x) && (slots == nullptr || apart(written, *slots)));
  Tensor h;
  const int status = unlocked([&] {
    h = make({B, H}, x->scalar_type(), *p);
    const int64_t st[3] = {gate->stride(0), x->stride(0), H};
    return b200_linear_recurrence_step_async_(gate->data_ptr(), x->data_ptr(), dtype, form, st, ptr<float>(state),
                                              ptr<float>(next ? next : state), ptr<int32_t>(slots), int(S), int(B),
                                              int(H), h.data_ptr(), p->stream);
  });
  return done(status, "linear_recurrence_step", h);
  END
}

// ------------------------------------------------------------------------------ token log-probs
struct Logits {
  int64_t B, T, V, st[4];
};
bool logits_ok(const Tensor& x, const Tensor& token, const Place& p, Logits* q) {
  const int64_t d = x.dim();
  if ((d != 2 && d != 3) || !rows(x, p, x.scalar_type(), d) || token.scalar_type() != at::kLong ||
      token.device() != p.device || token.sizes() != x.sizes().slice(0, d - 1))
    return false;
  q->V = x.size(-1);
  if (d == 2)
    *q = Logits{1, x.size(0), q->V, {0, x.stride(0), 0, token.stride(0)}};
  else
    *q = Logits{x.size(0), x.size(1), q->V, {x.stride(0), x.stride(1), token.stride(0), token.stride(1)}};
  return q->B * q->T <= kMax && q->V <= kMax;
}

// logprob(logits, token, temperature, entropy, train) -> (log_prob, entropy or None, stats or None)
PyObject* logprob(PyObject*, PyObject* const* a, Py_ssize_t n) {
  BEGIN
  const Tensor *x, *token;
  ORDINARY(n == 5 && (x = tensor(a[0])) && (token = tensor(a[1])) && PyFloat_CheckExact(a[2]));
  std::optional<Place> p;
  Logits q;
  const int dtype = code_of(*x);
  const double temperature = PyFloat_AS_DOUBLE(a[2]);
  ORDINARY(dtype >= 0 && temperature >= 1e-30 && temperature <= 1e30 && place_of(*x, &p) && logits_ok(*x, *token, *p, &q));
  Tensor lp, ent, stats;
  const bool entropy = a[3] == Py_True, train = a[4] == Py_True;
  const int status = unlocked([&] {
    lp = make(token->sizes(), at::kFloat, *p);
    if (entropy) ent = make(token->sizes(), at::kFloat, *p);
    if (train) {
      at::DimVector shape(token->sizes().begin(), token->sizes().end());
      shape.push_back(3);
      stats = make(shape, at::kFloat, *p);
    }
    return b200_token_logprob_async_(x->data_ptr(), dtype, q.st, ptr<int64_t>(token), int(q.B), int(q.T), int(q.V),
                                     temperature, ptr<float>(&lp), ptr<float>(&ent), ptr<float>(&stats), p->stream);
  });
  return done(status, "token_logprob", lp, ent, stats);
  END
}

// logprob_backward(logits, token, stats, grad_log_prob, grad_entropy, temperature) -> (grad_logits,)
PyObject* logprob_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  BEGIN
  const Tensor *x, *token, *stats, *gl, *ge;
  ORDINARY(n == 6 && (x = tensor(a[0])) && (token = tensor(a[1])) && (stats = tensor(a[2])) && (gl = tensor(a[3])) &&
           optional_tensor(a[4], &ge) && PyFloat_CheckExact(a[5]));
  std::optional<Place> p;
  Logits q;
  const int dtype = code_of(*x);
  const double temperature = PyFloat_AS_DOUBLE(a[5]);
  ORDINARY(dtype >= 0 && temperature >= 1e-30 && temperature <= 1e30 && place_of(*x, &p) && logits_ok(*x, *token, *p, &q));
  at::DimVector shape(token->sizes().begin(), token->sizes().end());
  shape.push_back(3);
  ORDINARY(dense(*stats, *p, at::kFloat, shape) && dense(*gl, *p, at::kFloat, token->sizes()) &&
           (ge == nullptr || dense(*ge, *p, at::kFloat, token->sizes())));
  Tensor out;
  const int status = unlocked([&] {
    out = make(x->sizes(), x->scalar_type(), *p);
    return b200_token_logprob_backward_async_(x->data_ptr(), dtype, q.st, ptr<int64_t>(token), ptr<float>(stats),
                                              ptr<float>(gl), ptr<float>(ge), int(q.B), int(q.T), int(q.V), temperature,
                                              out.data_ptr(), p->stream);
  });
  return done(status, "token_logprob_backward", out);
  END
}

// ----------------------------------------------------------------- policy and preference losses
// The numbers of an options tuple that ops.py has checked.
bool numbers(PyObject* t, double* v, Py_ssize_t n) {
  if (!PyTuple_CheckExact(t) || PyTuple_GET_SIZE(t) != n) return false;
  for (Py_ssize_t i = 0; i < n; ++i) v[i] = PyFloat_AsDouble(PyTuple_GET_ITEM(t, i));
  return true;
}

// policy(log_prob, old, advantage, mask, ref, entropy, options, want_grad, want_grad_entropy)
//   -> (outputs, grad_log_prob or None, grad_entropy or None)
PyObject* policy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  BEGIN
  const Tensor *lp, *old, *adv, *mask, *ref, *ent;
  double o[8];
  ORDINARY(n == 9 && (lp = tensor(a[0])) && optional_tensor(a[1], &old) && (adv = tensor(a[2])) &&
           optional_tensor(a[3], &mask) && optional_tensor(a[4], &ref) && optional_tensor(a[5], &ent) &&
           numbers(a[6], o, 8));
  std::optional<Place> p;
  ORDINARY(place_of(*lp, &p) && rows(*lp, *p, at::kFloat, 2));
  const int64_t B = lp->size(0), T = lp->size(1);
  const bool per_row = adv->dim() == 1;
  ORDINARY(B <= kMax && T <= kMax && stream_ok(old, *p, at::kFloat, B, T) && stream_ok(mask, *p, at::kBool, B, T) &&
           stream_ok(ref, *p, at::kFloat, B, T) && stream_ok(ent, *p, at::kFloat, B, T));
  ORDINARY(per_row ? adv->scalar_type() == at::kFloat && adv->device() == p->device && adv->size(0) == B
                   : stream_ok(adv, *p, at::kFloat, B, T));
  const int64_t bytes = b200_policy_loss_workspace_bytes_(int(B), int(T));
  const Tensor* ws = nullptr;
  ORDINARY(bytes == 0 || (ws = scratch(kPolicy, bytes, *p)) != nullptr);
  if (old == nullptr) old = lp;
  Tensor out, grad, ge;
  const bool want_grad = a[7] == Py_True, want_grad_entropy = a[8] == Py_True;
  const int status = unlocked([&] {
    out = make({8}, at::kFloat, *p);
    if (want_grad) grad = make({B, T}, at::kFloat, *p);
    if (want_grad_entropy) ge = make({B, T}, at::kFloat, *p);
    const int64_t st[7] = {lp->stride(0),   old->stride(0),  adv->stride(0), per_row ? 0 : 1,
                           row_stride(ref), row_stride(ent), row_stride(mask)};
    return b200_policy_loss_async_(ptr<float>(lp), ptr<float>(old), ptr<float>(adv), ptr<float>(ref), ptr<float>(ent),
                                   ptr<uint8_t>(mask), st, int(B), int(T), o[0], o[1], o[2], o[3], int(o[4]), o[5],
                                   int(o[6]), o[7], ptr<float>(&out), ptr<float>(&grad), ptr<float>(&ge), at_(ws),
                                   ws ? ws->numel() : 0, p->stream);
  });
  return done(status, "policy_loss", out, grad, ge);
  END
}

// preference(chosen, rejected, ref_chosen, ref_rejected, chosen_mask, rejected_mask, options, average, want_chosen,
//            want_rejected) -> (outputs, reward_chosen, reward_rejected, grad_chosen or None, grad_rejected or None)
PyObject* preference(PyObject*, PyObject* const* a, Py_ssize_t n) {
  BEGIN
  const Tensor *c, *r, *fc, *fr, *mc, *mr;
  double o[4];
  ORDINARY(n == 10 && (c = tensor(a[0])) && (r = tensor(a[1])) && optional_tensor(a[2], &fc) &&
           optional_tensor(a[3], &fr) && optional_tensor(a[4], &mc) && optional_tensor(a[5], &mr) &&
           numbers(a[6], o, 4) && (fc == nullptr) == (fr == nullptr));
  std::optional<Place> p;
  ORDINARY(place_of(*c, &p) && rows(*c, *p, at::kFloat, 2) && rows(*r, *p, at::kFloat, 2) && c->size(0) == r->size(0));
  const int64_t B = c->size(0), Tc = c->size(1), Tr = r->size(1);
  ORDINARY(B <= kMax && Tc <= kMax && Tr <= kMax && stream_ok(fc, *p, at::kFloat, B, Tc) &&
           stream_ok(fr, *p, at::kFloat, B, Tr) && stream_ok(mc, *p, at::kBool, B, Tc) &&
           stream_ok(mr, *p, at::kBool, B, Tr));
  const Tensor* ws = scratch(kPreference, b200_preference_loss_workspace_bytes_(int(B)), *p);
  ORDINARY(ws != nullptr);
  Tensor out, rc, rr, gc, gr;
  const bool average = a[7] == Py_True, want_chosen = a[8] == Py_True, want_rejected = a[9] == Py_True;
  const int status = unlocked([&] {
    out = make({3}, at::kFloat, *p), rc = make({B}, at::kFloat, *p), rr = make({B}, at::kFloat, *p);
    if (want_chosen) gc = make({B, Tc}, at::kFloat, *p);
    if (want_rejected) gr = make({B, Tr}, at::kFloat, *p);
    const int64_t st[6] = {c->stride(0),   r->stride(0),   row_stride(fc),
                           row_stride(fr), row_stride(mc), row_stride(mr)};
    return b200_preference_loss_async_(ptr<float>(c), ptr<float>(r), ptr<float>(fc), ptr<float>(fr), ptr<uint8_t>(mc),
                                       ptr<uint8_t>(mr), st, int(B), int(Tc), int(Tr), o[0], int(o[1]), o[2], o[3],
                                       average, ptr<float>(&out), ptr<float>(&rc), ptr<float>(&rr), ptr<float>(&gc),
                                       ptr<float>(&gr), at_(ws), ws->numel(), p->stream);
  });
  return done(status, "preference_loss", out, rc, rr, gc, gr);
  END
}

// init(path of the library, OpError, torch's version): ImportError for another torch than the one built for.
PyObject* init(PyObject*, PyObject* args) {
  const char *path, *version;
  PyObject* error;
  if (!PyArg_ParseTuple(args, "sOs", &path, &error, &version)) return nullptr;
  const size_t n = strlen(TORCH_VERSION);
  if (strncmp(version, TORCH_VERSION, n) != 0 || (version[n] != '\0' && version[n] != '+')) {
    PyErr_Format(PyExc_ImportError, "_calls was built for torch %s, not %s", TORCH_VERSION, version);
    return nullptr;
  }
  void* lib = dlopen(path, RTLD_NOW | RTLD_LOCAL);
  if (lib == nullptr) {
    PyErr_Format(PyExc_OSError, "%s", dlerror());
    return nullptr;
  }
  bool ok = true;
#define FIND(name) ok = (name##_ = reinterpret_cast<decltype(&::name)>(dlsym(lib, #name))) != nullptr && ok
  FIND(b200_status_string);
  FIND(b200_linear_recurrence_checkpoint_bytes);
  FIND(b200_linear_recurrence_workspace_bytes);
  FIND(b200_linear_recurrence_async);
  FIND(b200_linear_recurrence_backward_async);
  FIND(b200_linear_recurrence_step_async);
  FIND(b200_token_logprob_async);
  FIND(b200_token_logprob_backward_async);
  FIND(b200_policy_loss_workspace_bytes);
  FIND(b200_policy_loss_async);
  FIND(b200_preference_loss_workspace_bytes);
  FIND(b200_preference_loss_async);
  if (!ok) {
    PyErr_Format(PyExc_OSError, "%s lacks an entry point", path);
    return nullptr;
  }
  Py_INCREF(error);
  g_error = error;
  Py_RETURN_NONE;
}

template <typename F>
PyMethodDef fast(const char* name, F f) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr};
}

}  // namespace

PyMODINIT_FUNC PyInit__calls() {
  static PyMethodDef methods[] = {{"init", init, METH_VARARGS, nullptr},
                                  fast("recurrence", recurrence),
                                  fast("recurrence_backward", recurrence_backward),
                                  fast("recurrence_step", recurrence_step),
                                  fast("logprob", logprob),
                                  fast("logprob_backward", logprob_backward),
                                  fast("policy", policy),
                                  fast("preference", preference),
                                  {nullptr, nullptr, 0, nullptr}};
  static PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods};
  return PyModule_Create(&module);
}
