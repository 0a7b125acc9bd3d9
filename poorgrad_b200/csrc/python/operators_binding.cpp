// operators_binding.cpp -- the device operators of topos_b200.h on torch tensors, for
// poorgrad_b200/operators.py: checks of the arguments, outputs from torch's allocator on the
// current stream, one call of the C ABI.  Native because the checks and allocations of a small call
// cost more host time than its kernel takes: through ctypes a one-token scan took 15 us.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <sstream>

#include "../../../include/topos_b200.h"

namespace {

using at::IntArrayRef;
using at::ScalarType;
using at::Tensor;

PyObject* g_backend_error = nullptr;  // poorgrad_b200.backend.BackendError

[[noreturn]] void refuse(const std::string& why) {
  PyErr_SetString(PyExc_ValueError, why.c_str());
  throw python_error();
}
void need(bool condition, const char* why) {
  if (!condition) refuse(why);
}
void checked(int code, const char* entry) {
  if (code == TB_OK) return;
  if (!g_backend_error) {
    PyErr_Format(PyExc_RuntimeError, "%s: %s", entry, tb_last_error());
    throw python_error();
  }
  if (PyObject* error = PyObject_CallFunction(g_backend_error, "is", code, entry)) {
    PyErr_SetObject(g_backend_error, error);
    Py_DECREF(error);
  }
  throw python_error();
}

bool given(PyObject* o) { return o != Py_None; }
const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + ": a tensor is expected");
  return THPVariable_Unpack(o);
}

// What the arrays of one call share.
struct Arrays {
  at::Device device{at::kCPU};
  ScalarType type{};
  int64_t element = 0;

  Arrays(const Tensor& first, const char* name) : device(first.device()), type(first.scalar_type()) {
    if (!device.is_cuda() || (type != at::kFloat && type != at::kBFloat16))
      refuse(std::string(name) + ": a float32 or bfloat16 CUDA tensor is expected");
    element = type == at::kFloat ? TB_ELEMENT_F32 : TB_ELEMENT_BF16;
  }
  [[noreturn]] void unfit(const Tensor& t, const char* name, ScalarType want, IntArrayRef sizes,
                          const char* more) const {
    std::ostringstream s;
    s << name << ": expected " << want << " " << sizes << " on " << device << ", " << more << "; got "
      << t.scalar_type() << " " << t.sizes() << " with strides " << t.strides() << " on " << t.device();
    refuse(s.str());
  }
  // A large array: the call's type and device, this shape, stride 1 along the last axis.
  void* rows(const Tensor& t, const char* name, IntArrayRef sizes) const {
    if (t.scalar_type() != type || t.device() != device || t.sizes() != sizes ||
        (sizes.back() > 1 && t.strides().back() != 1))
      unfit(t, name, type, sizes, "stride 1 along the last axis");
    return t.data_ptr();
  }
  // A contiguous 32-bit array.
  template <typename W>
  W* words(const Tensor& t, const char* name, IntArrayRef sizes) const {
    const ScalarType want = std::is_same_v<W, float> ? at::kFloat : at::kInt;
    if (t.scalar_type() != want || t.device() != device || t.sizes() != sizes || !t.is_contiguous())
      unfit(t, name, want, sizes, "contiguous");
    return (W*)t.data_ptr();
  }
  template <typename W>
  W* words(PyObject* o, const char* name, IntArrayRef sizes) const {
    return given(o) ? words<W>(tensor(o, name), name, sizes) : nullptr;
  }
  Tensor made(IntArrayRef sizes, ScalarType t) const {
    return Tensor(at::detail::empty_cuda(sizes, t, device, std::nullopt));
  }
  // A new array in the order of t's axes, the last one innermost.
  Tensor like(const Tensor& t) const {
    if (!t.is_contiguous() && t.is_non_overlapping_and_dense() && t.strides().back() == 1) {
      Tensor same = at::empty_like(t);
      if (same.strides().back() == 1) return same;
    }
    return made(t.sizes(), type);
  }
  Tensor out(PyObject* o, const char* name, const Tensor& as) const {
    return given(o) ? tensor(o, name) : like(as);
  }
  void* stream() const { return (void*)c10::cuda::getCurrentCUDAStream(device.index()).stream(); }
};

// ------------------------------------------------- arrays that a call writes
// The bytes of an array, from the first to behind the last.
struct Place {
  const Tensor& t;
  const char *begin, *end;
  explicit Place(const Tensor& t) : t(t), begin((const char*)t.const_data_ptr()), end(begin) {
    if (t.numel() == 0) return;
    int64_t reach = 1;
    for (int64_t i = 0; i < t.dim(); ++i) reach += (t.size(i) - 1) * t.stride(i);
    end += reach * (int64_t)t.element_size();
  }
};
// Whether an element of the one, `apart` elements behind the other's first, is one of the other: strides
// `s`, `n` steps forwards of the one and `m` of the other, from axis i on.
bool step_onto(int64_t apart, int i, const int64_t* s, const int64_t* n, const int64_t* m, int axes) {
  if (i == axes) return apart == 0;
  int64_t back = 0, forth = 0;  // what the axes behind this one reach
  for (int j = i + 1; j < axes; ++j) back += m[j] * s[j], forth += n[j] * s[j];
  // steps k of this axis that leave the rest within reach: -back <= apart - k s <= forth
  const auto down = [](int64_t a, int64_t b) { return a >= 0 ? a / b : -((-a + b - 1) / b); };
  const int64_t from = std::max(-m[i], -down(forth - apart, s[i])), to = std::min(n[i], down(apart + back, s[i]));
  for (int64_t k = from; k <= to; ++k)
    if (step_onto(apart - k * s[i], i + 1, s, n, m, axes)) return true;
  return false;
}
// Whether two arrays of the same axes share an element.  Arrays that lie in one another's gaps with
// strides of their own are taken to share none.
bool meet(const Place& a, const Place& b) {
  if (a.begin >= b.end || b.begin >= a.end) return false;
  constexpr int kAxes = 4;
  const int64_t size = a.t.element_size();
  if (a.t.dim() != b.t.dim() || a.t.dim() > kAxes || b.t.element_size() != size || (b.begin - a.begin) % size)
    return true;
  int64_t s[kAxes], n[kAxes], m[kAxes];
  int axes = 0;
  for (int64_t i = 0; i < a.t.dim(); ++i) {
    const int64_t steps = a.t.size(i) - 1, others = b.t.size(i) - 1;
    if (steps == 0 && others == 0) continue;
    const int64_t stride = steps ? a.t.stride(i) : b.t.stride(i);
    if ((steps && others && a.t.stride(i) != b.t.stride(i)) || stride <= 0) return a.begin == b.begin;
    int at = axes++;
    for (; at > 0 && s[at - 1] < stride; --at) s[at] = s[at - 1], n[at] = n[at - 1], m[at] = m[at - 1];
    s[at] = stride, n[at] = steps, m[at] = others;
  }
  return step_onto((b.begin - a.begin) / size, 0, s, n, m, axes);
}
bool same(const Place& a, const Place& b) {
  if (a.begin != b.begin || a.t.sizes() != b.t.sizes()) return false;
  for (int64_t i = 0; i < a.t.dim(); ++i)
    if (a.t.size(i) > 1 && a.t.stride(i) != b.t.stride(i)) return false;
  return true;
}
// An output may not share memory with another one or with an input; with an input that it may take
// the place of, it shares all of it.
void apart(const Place& a, const char* name, const Place& b, const char* other, bool in_place = false) {
  if (meet(a, b) && !(in_place && same(a, b)))
    refuse(std::string(name) + " shares memory with " + other + (in_place ? ", but is not the same array" : ""));
}
// What autograd has to know of an array that the caller gave and a call has written.
void written(PyObject* o) {
  if (!o || !THPVariable_Check(o)) return;
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

PyObject* wrapped(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* wrapped_or_none(const Tensor& t) {
  if (t.defined()) return wrapped(t);
  Py_RETURN_NONE;
}
template <typename... T>
PyObject* tuple_of(const T&... t) {
  PyObject* r = PyTuple_New(sizeof...(T));
  if (!r) throw python_error();
  Py_ssize_t i = 0;
  ((PyTuple_SET_ITEM(r, i++, wrapped_or_none(t))), ...);
  return r;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
int64_t whole(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
void arguments(Py_ssize_t got, Py_ssize_t want) {
  if (got == want) return;
  PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, got);
  throw python_error();
}

// ------------------------------------------------------------------ gated scan
// The extents of a call by its first array; `states`: the shape of its states.
struct ScanExtents {
  bool packed;
  int64_t states[2];
  ScanExtents(tb_scan_desc& d, const Tensor& x, PyObject* offsets) : packed(given(offsets)) {
    if (packed) {
      need(x.dim() == 2, "a packed batch is [rows, channels]");
      const Tensor& o = tensor(offsets, "offsets");
      need(o.dim() == 1 && o.size(0) >= 2, "offsets: expected sequences + 1 row numbers");
      d.batch = 1;
      d.sequences = o.size(0) - 1;
    } else {
      need(x.dim() == 3, "expected [batch, length, channels], or packed [rows, channels] with offsets");
      d.batch = x.size(0);
      d.sequences = 0;
    }
    d.length = x.size(-2);
    d.channels = x.size(-1);
    states[0] = packed ? d.sequences : d.batch;
    states[1] = d.channels;
  }
  void strides(const Tensor& t, int64_t s[2]) const {
    s[0] = packed ? 0 : t.stride(0);
    s[1] = t.stride(-2);
  }
};
Tensor scan_scratch(tb_scan_desc& d, const Arrays& a) {
  d.workspace_bytes = tb_gated_scan_workspace(d.batch, d.length, d.channels);
  if (!d.workspace_bytes) return {};
  Tensor scratch = a.made({d.workspace_bytes}, at::kByte);
  d.workspace = scratch.data_ptr();
  return scratch;
}

// gate, x, form, state, offsets, out, final_state
PyObject* gated_scan(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 7);
  const Tensor &gate = tensor(v[0], "gate"), &x = tensor(v[1], "x");
  const Arrays a(x, "x");
  tb_scan_desc d = {};
  const ScanExtents e(d, x, v[4]);
  const c10::cuda::CUDAGuard guard(a.device);
  const Tensor out = a.out(v[5], "out", x);
  const Tensor final_state = given(v[6]) ? tensor(v[6], "final_state") : a.made(e.states, at::kFloat);
  d.element = a.element;
  d.form = whole(v[2]);
  d.gate = a.rows(gate, "gate", x.sizes());
  d.x = a.rows(x, "x", x.sizes());
  d.h = a.rows(out, "out", x.sizes());
  d.offsets = a.words<int32_t>(v[4], "offsets", {d.sequences + 1});
  d.state = a.words<float>(v[3], "state", e.states);
  d.final_state = a.words<float>(final_state, "final_state", e.states);
  e.strides(gate, d.gate_strides);
  e.strides(x, d.x_strides);
  e.strides(out, d.h_strides);
  if (given(v[5]) || given(v[6])) {
    const Place to(out), last(final_state), from_gate(gate), from_x(x);
    apart(to, "out", from_gate, "gate", true);
    apart(to, "out", from_x, "x", true);
    apart(to, "out", last, "final_state");
    apart(last, "final_state", from_gate, "gate");
    apart(last, "final_state", from_x, "x");
    if (given(v[3])) {
      const Place state(tensor(v[3], "state"));
      apart(last, "final_state", state, "state", true);
      apart(to, "out", state, "state");
    }
  }
  d.clear = given(v[5]) ? 0 : TB_SCAN_CLEAR_H;  // new arrays hold nothing to leave as it was
  const Tensor scratch = scan_scratch(d, a);
  checked(tb_gated_scan(&d, a.stream()), "tb_gated_scan");
  written(v[5]);
  written(v[6]);
  return tuple_of(out, final_state);
  END_HANDLE_TH_ERRORS
}

// dh, gate, x, h, form, state, offsets, dfinal, dgate, dx
PyObject* gated_scan_backward(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 10);
  const Tensor &dh = tensor(v[0], "dh"), &gate = tensor(v[1], "gate"), &h = tensor(v[3], "h");
  const Arrays a(dh, "dh");
  tb_scan_desc d = {};
  const ScanExtents e(d, dh, v[6]);
  const c10::cuda::CUDAGuard guard(a.device);
  const Tensor dgate = a.out(v[8], "dgate", dh), dx = a.out(v[9], "dx", dh);
  const Tensor dstate = a.made(e.states, at::kFloat);
  d.element = a.element;
  d.form = whole(v[4]);
  if (given(v[2]) || d.form != TB_SCAN_DIRECT) {  // the direct form does not read x
    const Tensor& x = tensor(v[2], "x");
    d.x = a.rows(x, "x", dh.sizes());
    e.strides(x, d.x_strides);
  }
  d.gate = a.rows(gate, "gate", dh.sizes());
  d.h = a.rows(h, "h", dh.sizes());
  d.dh = a.rows(dh, "dh", dh.sizes());
  d.dgate = a.rows(dgate, "dgate", dh.sizes());
  d.dx = a.rows(dx, "dx", dh.sizes());
  d.offsets = a.words<int32_t>(v[6], "offsets", {d.sequences + 1});
  d.state = a.words<float>(v[5], "state", e.states);
  d.dfinal = a.words<float>(v[7], "dfinal", e.states);
  d.dstate = (float*)dstate.data_ptr();
  e.strides(gate, d.gate_strides);
  e.strides(h, d.h_strides);
  e.strides(dh, d.dh_strides);
  e.strides(dgate, d.dgate_strides);
  e.strides(dx, d.dx_strides);
  if (given(v[8]) || given(v[9])) {
    const Place to_gate(dgate), to_x(dx), from_dh(dh), from_gate(gate), from_h(h);
    apart(to_gate, "dgate", to_x, "dx");
    // a row of h is read for the next step's gradient too
    apart(to_gate, "dgate", from_h, "h");
    apart(to_x, "dx", from_h, "h");
    apart(to_gate, "dgate", from_dh, "dh", true);
    apart(to_x, "dx", from_dh, "dh", true);
    apart(to_gate, "dgate", from_gate, "gate", true);
    apart(to_x, "dx", from_gate, "gate", true);
    if (d.form != TB_SCAN_DIRECT) {
      const Place from_x(tensor(v[2], "x"));
      apart(to_gate, "dgate", from_x, "x", true);
      apart(to_x, "dx", from_x, "x", true);
    }
    for (int i : {5, 7})
      if (given(v[i])) {
        const Place from(tensor(v[i], "state"));
        apart(to_gate, "dgate", from, i == 5 ? "state" : "dfinal");
        apart(to_x, "dx", from, i == 5 ? "state" : "dfinal");
      }
  }
  d.clear = (given(v[8]) ? 0 : TB_SCAN_CLEAR_DGATE) | (given(v[9]) ? 0 : TB_SCAN_CLEAR_DX);
  const Tensor scratch = scan_scratch(d, a);
  checked(tb_gated_scan_backward(&d, a.stream()), "tb_gated_scan_backward");
  written(v[8]);
  written(v[9]);
  return tuple_of(dgate, dx, dstate);
  END_HANDLE_TH_ERRORS
}

// ----------------------------------------------------------------- head rotate
// Heads [batch, length, heads, dim], or [tokens, heads, dim] as one batch row.
void head_strides(const Tensor& t, int64_t s[3]) {
  s[0] = t.dim() == 4 ? t.stride(0) : 0;
  s[1] = t.stride(-3);
  s[2] = t.stride(-2);
}
// q, k, table, positions, q_weight, k_weight, epsilon, style, q_out, k_out
struct RotateCall {
  Arrays a;
  const Tensor &q, &k;
  c10::cuda::CUDAGuard guard;
  Tensor q_out, k_out;
  tb_rotate_desc d = {};
  explicit RotateCall(PyObject* const* v)
      : a(tensor(v[0], "q"), "q"), q(THPVariable_Unpack(v[0])), k(tensor(v[1], "k")), guard(a.device) {
    need((q.dim() == 3 || q.dim() == 4) && k.dim() == q.dim(),
         "q, k: expected [tokens, heads, dim] or [batch, length, heads, dim]");
    const Tensor& table = tensor(v[2], "table");
    need(table.dim() == 2, "table: expected [positions, turned]");
    q_out = a.out(v[8], "q_out", q);
    k_out = a.out(v[9], "k_out", k);
    d.element = a.element;
    d.style = whole(v[7]);
    d.batch = q.dim() == 4 ? q.size(0) : 1;
    d.length = q.size(-3);
    d.q_heads = q.size(-2);
    d.k_heads = k.size(-2);
    d.dim = q.size(-1);
    d.turned = table.size(1);
    d.table_rows = table.size(0);
    d.epsilon = number(v[6]);
    d.q = a.rows(q, "q", q.sizes());
    d.q_out = a.rows(q_out, "q_out", q.sizes());
    k_sizes = q.sizes().vec();
    k_sizes[q.dim() - 2] = d.k_heads;
    d.k = a.rows(k, "k", k_sizes);
    d.k_out = a.rows(k_out, "k_out", k_sizes);
    d.table = a.words<float>(table, "table", table.sizes());
    if (given(v[3])) {
      const Tensor& p = tensor(v[3], "positions");
      d.positions = p.dim() == 1 && q.dim() == 3
                        ? a.words<int32_t>(p, "positions", {d.length})
                        : a.words<int32_t>(p, "positions", {d.batch, d.length});
    }
    d.q_weight = a.words<float>(v[4], "q_weight", {d.dim});
    d.k_weight = a.words<float>(v[5], "k_weight", {d.dim});
    head_strides(q, d.q_strides);
    head_strides(k, d.k_strides);
    head_strides(q_out, d.q_out_strides);
    head_strides(k_out, d.k_out_strides);
  }
  std::vector<int64_t> k_sizes;
  // No output in the place of anything but its own inputs.
  void outputs_apart(PyObject* const* v, const Tensor* dq = nullptr, const Tensor* dk = nullptr) const {
    if (!given(v[8]) && !given(v[9])) return;
    const Place to_q(q_out), to_k(k_out), from_q(q), from_k(k);
    apart(to_q, "q_out", to_k, "k_out");
    apart(to_q, "q_out", from_q, "q", true);
    apart(to_q, "q_out", from_k, "k");
    apart(to_k, "k_out", from_k, "k", true);
    apart(to_k, "k_out", from_q, "q");
    if (dq) {
      const Place grad_q(*dq), grad_k(*dk);
      apart(to_q, "q_out", grad_q, "dq", true);
      apart(to_q, "q_out", grad_k, "dk");
      apart(to_k, "k_out", grad_k, "dk", true);
      apart(to_k, "k_out", grad_q, "dq");
    }
  }
};
PyObject* head_rotate(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 10);
  const RotateCall call(v);
  call.outputs_apart(v);
  checked(tb_head_rotate(&call.d, call.a.stream()), "tb_head_rotate");
  written(v[8]);
  written(v[9]);
  return tuple_of(call.q_out, call.k_out);
  END_HANDLE_TH_ERRORS
}
// those, then dq, dk, weights
PyObject* head_rotate_backward(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 13);
  RotateCall call(v);
  tb_rotate_desc& d = call.d;
  const Tensor &dq = tensor(v[10], "dq"), &dk = tensor(v[11], "dk");
  d.dq = call.a.rows(dq, "dq", call.q.sizes());
  d.dk = call.a.rows(dk, "dk", call.k_sizes);
  head_strides(dq, d.dq_strides);
  head_strides(dk, d.dk_strides);
  call.outputs_apart(v, &dq, &dk);
  Tensor dq_weight, dk_weight, scratch;
  if (v[12] == Py_True) {
    dq_weight = call.a.made({d.dim}, at::kFloat);
    dk_weight = call.a.made({d.dim}, at::kFloat);
    d.workspace_bytes = tb_head_rotate_workspace(d.dim);
    scratch = call.a.made({d.workspace_bytes}, at::kByte);
    d.dq_weight = (float*)dq_weight.data_ptr();
    d.dk_weight = (float*)dk_weight.data_ptr();
    d.workspace = scratch.data_ptr();
  }
  checked(tb_head_rotate_backward(&d, call.a.stream()), "tb_head_rotate_backward");
  written(v[8]);
  written(v[9]);
  return tuple_of(call.q_out, call.k_out, dq_weight, dk_weight);
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------------- losses
const Tensor& logits_of(PyObject* o) {
  const Tensor& t = tensor(o, "logits");
  need(t.dim() == 2, "logits: expected [rows, vocab]");
  return t;
}
// True, False, None, or the array to write.
Tensor gradient_of(PyObject* o, const Tensor& logits, const Arrays& a) {
  if (o == Py_False || o == Py_None) return {};
  const Tensor t = o == Py_True ? a.like(logits) : tensor(o, "gradient");
  a.rows(t, "gradient", logits.sizes());
  if (o != Py_True) apart(Place(t), "gradient", Place(logits), "logits", true);
  return t;
}

// logits, targets, scale
PyObject* token_logp(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 3);
  const Tensor& logits = logits_of(v[0]);
  const Arrays a(logits, "logits");
  const int64_t rows = logits.size(0);
  const void* z = a.rows(logits, "logits", logits.sizes());
  const int32_t* targets = a.words<int32_t>(tensor(v[1], "targets"), "targets", {rows});
  const c10::cuda::CUDAGuard guard(a.device);
  const Tensor logp = a.made({rows}, at::kFloat);
  checked(tb_token_logp(a.element, z, logits.stride(0), targets, rows, logits.size(1), number(v[2]),
                        (float*)logp.data_ptr(), a.stream()),
          "tb_token_logp");
  return wrapped(logp);
  END_HANDLE_TH_ERRORS
}

// logits, targets, old_logp, advantages, weights, ref_logp, clip_low, clip_high, kl, scale, gradient
PyObject* policy_loss(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 11);
  const Tensor& logits = logits_of(v[0]);
  const Arrays a(logits, "logits");
  const int64_t rows = logits.size(0);
  tb_policy_desc d = {};
  d.element = a.element;
  d.rows = rows;
  d.vocab = logits.size(1);
  d.logits = a.rows(logits, "logits", logits.sizes());
  d.logits_stride = logits.stride(0);
  d.targets = a.words<int32_t>(tensor(v[1], "targets"), "targets", {rows});
  d.old_logp = a.words<float>(tensor(v[2], "old_logp"), "old_logp", {rows});
  d.advantages = a.words<float>(tensor(v[3], "advantages"), "advantages", {rows});
  d.weights = a.words<float>(tensor(v[4], "weights"), "weights", {rows});
  d.ref_logp = a.words<float>(v[5], "ref_logp", {rows});
  d.clip_low = number(v[6]);
  d.clip_high = number(v[7]);
  d.kl = number(v[8]);
  d.scale = number(v[9]);
  need(!(d.kl > 0) || given(v[5]), "ref_logp is needed where kl is not 0");
  const c10::cuda::CUDAGuard guard(a.device);
  const Tensor gradient = gradient_of(v[10], logits, a);
  const Tensor loss = a.made({}, at::kFloat), token_loss = a.made({rows}, at::kFloat),
               logp = a.made({rows}, at::kFloat);
  if (gradient.defined()) {
    d.gradient = gradient.data_ptr();
    d.gradient_stride = gradient.stride(0);
  }
  d.loss = (float*)loss.data_ptr();
  d.token_loss = (float*)token_loss.data_ptr();
  d.logp = (float*)logp.data_ptr();
  checked(tb_policy_loss(&d, a.stream()), "tb_policy_loss");
  written(v[10]);
  return tuple_of(loss, token_loss, logp, gradient);
  END_HANDLE_TH_ERRORS
}

// logits, targets, offsets, ref_logp, beta, smoothing, weights, scale, gradient
PyObject* preference_loss(PyObject*, PyObject* const* v, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 9);
  const Tensor& logits = logits_of(v[0]);
  const Arrays a(logits, "logits");
  const Tensor& offsets = tensor(v[2], "offsets");
  need(offsets.dim() == 1 && offsets.size(0) >= 3 && offsets.size(0) % 2 == 1,
       "offsets: expected 2 pairs + 1 row numbers");
  const int64_t rows = logits.size(0), pairs = offsets.size(0) / 2;
  tb_preference_desc d = {};
  d.element = a.element;
  d.rows = rows;
  d.vocab = logits.size(1);
  d.pairs = pairs;
  d.logits = a.rows(logits, "logits", logits.sizes());
  d.logits_stride = logits.stride(0);
  d.targets = a.words<int32_t>(tensor(v[1], "targets"), "targets", {rows});
  d.offsets = a.words<int32_t>(offsets, "offsets", {2 * pairs + 1});
  d.ref_logp = a.words<float>(tensor(v[3], "ref_logp"), "ref_logp", {rows});
  d.beta = number(v[4]);
  d.smoothing = number(v[5]);
  d.weights = a.words<float>(v[6], "weights", {pairs});
  d.scale = number(v[7]);
  const c10::cuda::CUDAGuard guard(a.device);
  const Tensor gradient = gradient_of(v[8], logits, a);
  const Tensor loss = a.made({}, at::kFloat), ratios = a.made({2 * pairs}, at::kFloat),
               logp = a.made({rows}, at::kFloat);
  d.workspace_bytes = tb_preference_workspace(rows, pairs);
  const Tensor scratch = a.made({d.workspace_bytes}, at::kByte);
  if (gradient.defined()) {
    d.gradient = gradient.data_ptr();
    d.gradient_stride = gradient.stride(0);
  }
  d.loss = (float*)loss.data_ptr();
  d.ratios = (float*)ratios.data_ptr();
  d.logp = (float*)logp.data_ptr();
  d.workspace = scratch.data_ptr();
  d.clear = TB_PREFERENCE_CLEAR_LOGP | (v[8] == Py_True ? TB_PREFERENCE_CLEAR_GRADIENT : 0);
  checked(tb_preference_loss(&d, a.stream()), "tb_preference_loss");
  written(v[8]);
  return tuple_of(loss, ratios, logp, gradient);
  END_HANDLE_TH_ERRORS
}

PyObject* set_error(PyObject*, PyObject* error) {
  Py_INCREF(error);
  Py_XSETREF(g_backend_error, error);
  Py_RETURN_NONE;
}

#define TB_METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {TB_METHOD(gated_scan),
                         TB_METHOD(gated_scan_backward),
                         TB_METHOD(head_rotate),
                         TB_METHOD(head_rotate_backward),
                         TB_METHOD(token_logp),
                         TB_METHOD(policy_loss),
                         TB_METHOD(preference_loss),
                         {"set_error", set_error, METH_O, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_operators", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__operators() { return PyModule_Create(&module); }
