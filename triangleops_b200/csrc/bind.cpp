// bind.cpp — the Python face of the token block's operators (window_attn, gated_norm, rotary): a
// CPython extension that checks the tensors of a call, allocates its results and calls the C ABI.
//
// A call for one token takes the GPU 3 to 7 us; checks, allocations and a ctypes call in Python took
// 14 to 20 us around it, these functions take 5.6 to 7, the launch included.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/triangleops_b200.h"
#include "status.h"

namespace {

using at::Tensor;

// A refusal: an exception of a Python type, on its way to the interpreter.
struct Refused {};
[[noreturn]] void refuse(PyObject* type, const std::string& text) {
  PyErr_SetString(type, text.c_str());
  throw Refused();
}
void must(bool ok, const char* text) {
  if (!ok) refuse(PyExc_AssertionError, text);
}

// The statuses of the C ABI as the exceptions that the rest of the package raises for them.
void check(int code, const char* what) {
  if (code == TOPS_OK) return;
  PyObject* type = code == TOPS_ERR_SHAPE || code == TOPS_ERR_ALIGN ? PyExc_AssertionError
                   : code == TOPS_ERR_DTYPE || code == TOPS_ERR_ARG ? PyExc_ValueError
                                                                    : PyExc_RuntimeError;
  refuse(type, std::string(what) + ": " + tops_status_string(code) + " (status " + std::to_string(code) + ")");
}

const Tensor& tensor(PyObject* o) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string("expected a tensor, got ") + Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
Tensor maybe(PyObject* o) { return o == Py_None ? Tensor() : tensor(o); }
int64_t whole(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused();
  return v;
}
int flag(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Refused();
  return v;
}
double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refused();
  return v;
}

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return TOPS_F16;
    case at::kBFloat16: return TOPS_BF16;
    case at::kFloat: return TOPS_F32;
    default:
      refuse(PyExc_ValueError, std::string("unsupported IO dtype ") + at::toString(t.scalar_type()) +
                                   "; expected fp16, bf16 or fp32");
  }
}
void same_dtype(const Tensor& a, const Tensor& b, const char* what) {
  if (b.defined() && b.scalar_type() != a.scalar_type())
    refuse(PyExc_ValueError, std::string(what) + " must have one dtype, got " + at::toString(a.scalar_type()) + " and " +
                                 at::toString(b.scalar_type()));
}
void require_cuda(const Tensor& t) {
  if (!t.is_cuda())
    refuse(PyExc_RuntimeError, "triangleops_b200 runs only on CUDA (sm_100a) tensors; got a tensor on " +
                                   t.device().str() + ". There is no CPU fallback.");
}

Tensor empty(at::IntArrayRef shape, at::ScalarType type, const at::Device& dev) {
  return at::detail::empty_cuda(shape, type, dev, std::nullopt);
}
Tensor like(const Tensor& t) { return empty(t.sizes(), t.scalar_type(), t.device()); }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

PyObject* give(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
template <typename... Ts>
PyObject* give_tuple(const Ts&... ts) {
  PyObject* r = PyTuple_New(sizeof...(ts));
  if (r == nullptr) throw Refused();
  Py_ssize_t i = 0;
  (PyTuple_SET_ITEM(r, i++, give(ts)), ...);
  return r;
}

// ---------------------------------------------------------------------------
// windowed attention
// ---------------------------------------------------------------------------
// The tensor with contiguous channels (a copy where it has none).
Tensor rows(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

// As rows(), and where the tensor cores take the type and head size, with rows that their loads can
// follow: 16-byte aligned, none repeated by a stride of zero (one copy costs far less than the
// CUDA-core path that takes such rows as they are).
Tensor tiles(const Tensor& t0) {
  Tensor t = rows(t0);
  if (t.scalar_type() == at::kFloat || t.size(-1) % 8 != 0 || t.size(-1) > 128) return t;
  bool fits = reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i) fits = fits && (t.size(i) <= 1 || (t.stride(i) % 8 == 0 && t.stride(i) > 0));
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}

struct Attn {
  int dt;
  int64_t B, Nq, Nk, Hq, Hkv, D;
  Attn(const Tensor& q, const Tensor& k, const Tensor& v) {
    dt = dtype_code(q);
    must(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k and v must be (B, N, H, D)");
    B = q.size(0), Nq = q.size(1), Hq = q.size(2), D = q.size(3), Nk = k.size(1), Hkv = k.size(2);
    must(k.sizes() == v.sizes() && k.size(0) == B && k.size(3) == D, "k and v must be (B, Nk, Hkv, D) like q");
    must(Hkv > 0 && Hq % Hkv == 0, "the query heads must be a multiple of the key heads");
    must(Nk >= Nq, "the queries are the last Nq of the Nk tokens");
    same_dtype(q, k, "q, k and v");
    same_dtype(q, v, "q, k and v");
    must(q.device() == k.device() && q.device() == v.device(), "q, k and v must be on one device");
  }
  Tensor mask(PyObject* o, const Tensor& q) const {
    Tensor m = maybe(o);
    if (!m.defined()) return m;
    must(m.dim() == 2 && m.size(0) == B && m.size(1) == Nk, "mask must be (B, Nk)");
    must(m.device() == q.device(), "mask must be on the device of q");
    if (m.scalar_type() != at::kBool) m = m.ne(0);
    return m.contiguous();
  }
  float scale(PyObject* o) const { return static_cast<float>(o == Py_None ? 1.0 / std::sqrt(static_cast<double>(D)) : real(o)); }
};

struct Strides {
  int64_t s[9];
  Strides(const Tensor& q, const Tensor& k, const Tensor& v) {
    for (int i = 0; i < 3; ++i) s[i] = q.stride(i), s[3 + i] = k.stride(i), s[6 + i] = v.stride(i);
  }
};

// (q, k, v, mask, left, right, sinks, scale, out) -> (out, lse)
PyObject* window_attn_forward(PyObject* const* a) {
  Tensor q = tensor(a[0]), k = tensor(a[1]), v = tensor(a[2]);
  const Attn s(q, k, v);
  require_cuda(q);
  const c10::cuda::CUDAGuard guard(q.device());
  const Tensor m = s.mask(a[3], q);
  Tensor out = maybe(a[8]);
  if (out.defined())
    must(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.is_contiguous() &&
             out.device() == q.device(),
         "out must be like q, contiguous");
  else
    out = like(q);
  q = tiles(q), k = tiles(k), v = tiles(v);
  const Tensor lse = empty({s.B, s.Hq, s.Nq}, at::kFloat, q.device());
  check(tops_window_attn_forward(s.dt, s.B, s.Nq, s.Nk, s.Hq, s.Hkv, s.D, ptr(q), ptr(k), ptr(v), Strides(q, k, v).s,
                                 static_cast<const uint8_t*>(ptr(m)), whole(a[4]), whole(a[5]), whole(a[6]),
                                 s.scale(a[7]), out_ptr(out), static_cast<float*>(out_ptr(lse)), stream_of(q)),
        "tops_window_attn_forward");
  return give_tuple(out, lse);
}

// (dout, q, k, v, out, lse, mask, left, right, sinks, scale) -> (dq, dk, dv)
PyObject* window_attn_backward(PyObject* const* a) {
  Tensor dout = tensor(a[0]), q = tensor(a[1]), k = tensor(a[2]), v = tensor(a[3]), out = tensor(a[4]),
         lse = tensor(a[5]);
  const Attn s(q, k, v);
  must(dout.sizes() == q.sizes() && out.sizes() == q.sizes(), "dout and out must be like q");
  must(lse.dim() == 3 && lse.size(0) == s.B && lse.size(1) == s.Hq && lse.size(2) == s.Nq &&
           lse.scalar_type() == at::kFloat,
       "lse must be (B, Hq, Nq) fp32");
  same_dtype(q, dout, "q, dout and out");
  same_dtype(q, out, "q, dout and out");
  must(dout.device() == q.device() && out.device() == q.device() && lse.device() == q.device(),
       "dout, out and lse must be on the device of q");
  require_cuda(q);
  const c10::cuda::CUDAGuard guard(q.device());
  const Tensor m = s.mask(a[6], q);
  const int64_t left = whole(a[7]), right = whole(a[8]), sinks = whole(a[9]);
  const Tensor dq = like(q), dk = like(k), dv = like(k);
  q = tiles(q), k = tiles(k), v = tiles(v), dout = tiles(dout), out = out.contiguous(), lse = lse.contiguous();
  int64_t need = 0;
  check(tops_window_attn_backward_workspace_bytes(s.dt, s.B, s.Nq, s.Nk, s.Hq, s.Hkv, s.D, left, right, sinks, &need),
        "tops_window_attn_backward");
  const Tensor ws = empty({need < 16 ? 16 : need}, at::kByte, q.device());
  const int64_t ds[3] = {dout.stride(0), dout.stride(1), dout.stride(2)};
  check(tops_window_attn_backward(s.dt, s.B, s.Nq, s.Nk, s.Hq, s.Hkv, s.D, ptr(q), ptr(k), ptr(v), Strides(q, k, v).s,
                                  static_cast<const uint8_t*>(ptr(m)), left, right, sinks, s.scale(a[10]), ptr(dout), ds,
                                  ptr(out), static_cast<const float*>(ptr(lse)), out_ptr(ws), out_ptr(dq), out_ptr(dk),
                                  out_ptr(dv), stream_of(q)),
        "tops_window_attn_backward");
  return give_tuple(dq, dk, dv);
}

// Lengths as the kernels read them. A wider type's are brought into -1..N first (below and above it they
// all mean the same), where their low 32 bits could be any number.
Tensor lengths32(const Tensor& n, int64_t N) {
  if (n.scalar_type() == at::kInt) return n.contiguous();
  const bool wide = n.scalar_type() == at::kLong || n.is_floating_point();
  return (wide ? n.clamp(-1, N) : n).to(at::kInt).contiguous();
}

// (q, k_cache, v_cache, lengths, window, sinks, scale) -> out
PyObject* window_attn_decode(PyObject* const* a) {
  Tensor q = tensor(a[0]), k = tensor(a[1]), v = tensor(a[2]), n = tensor(a[3]);
  const int dt = dtype_code(q);
  must(q.dim() == 3, "q must be (B, Hq, D)");
  must(k.dim() == 4 && k.sizes() == v.sizes(), "the caches must be (B, N, Hkv, D)");
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2), N = k.size(1), Hkv = k.size(2);
  must(k.size(0) == B && k.size(3) == D, "the caches must be (B, N, Hkv, D) like q");
  must(Hkv > 0 && Hq % Hkv == 0, "the query heads must be a multiple of the key heads");
  same_dtype(q, k, "q and the caches");
  same_dtype(q, v, "q and the caches");
  must(k.device() == q.device() && v.device() == q.device() && n.device() == q.device(),
       "q, the caches and lengths must be on one device");
  must(n.dim() == 1 && n.size(0) == B, "lengths must be (B,)");
  const int64_t window = whole(a[4]), sinks = whole(a[5]);
  if (window < 1) refuse(PyExc_ValueError, "window must be a number of keys, at least 1, got " + std::to_string(window));
  const float scale = static_cast<float>(a[6] == Py_None ? 1.0 / std::sqrt(static_cast<double>(D)) : real(a[6]));
  require_cuda(q);
  const c10::cuda::CUDAGuard guard(q.device());
  q = rows(q), k = rows(k), v = rows(v), n = lengths32(n, N);
  const Tensor out = like(q);
  int64_t need = 0;
  check(tops_window_attn_decode_workspace_bytes(B, N, Hq, Hkv, D, window, sinks, &need), "tops_window_attn_decode");
  const Tensor ws = need > 0 ? empty({need}, at::kByte, q.device()) : Tensor();
  const int64_t st[8] = {q.stride(0), q.stride(1), k.stride(0), k.stride(1), k.stride(2),
                         v.stride(0), v.stride(1), v.stride(2)};
  check(tops_window_attn_decode(dt, B, N, Hq, Hkv, D, ptr(q), ptr(k), ptr(v), st, static_cast<const int32_t*>(ptr(n)),
                                window, sinks, scale, out_ptr(ws), out_ptr(out), stream_of(q)),
        "tops_window_attn_decode");
  return give(out);
}

// (k, v, k_cache, v_cache, lengths) -> None
PyObject* window_attn_store(PyObject* const* a) {
  Tensor k = tensor(a[0]), v = tensor(a[1]), n = tensor(a[4]);
  const Tensor kc = tensor(a[2]), vc = tensor(a[3]);
  const int dt = dtype_code(k);
  must(k.dim() == 3 && k.sizes() == v.sizes(), "k and v must be (B, Hkv, D)");
  const int64_t B = k.size(0), H = k.size(1), D = k.size(2);
  must(kc.dim() == 4 && kc.sizes() == vc.sizes() && kc.size(0) == B && kc.size(2) == H && kc.size(3) == D,
       "the caches must be (B, N, Hkv, D) like k and v");
  must(n.dim() == 1 && n.size(0) == B, "lengths must be (B,)");
  same_dtype(k, v, "k, v and the caches");
  same_dtype(k, kc, "k, v and the caches");
  same_dtype(k, vc, "k, v and the caches");
  must(v.device() == k.device() && kc.device() == k.device() && vc.device() == k.device() && n.device() == k.device(),
       "k, v, the caches and lengths must be on one device");
  require_cuda(k);
  const c10::cuda::CUDAGuard guard(k.device());
  k = rows(k), v = rows(v), n = lengths32(n, kc.size(1));
  const int64_t st[4] = {k.stride(0), k.stride(1), v.stride(0), v.stride(1)};
  int64_t ct[8];
  for (int i = 0; i < 4; ++i) ct[i] = kc.stride(i), ct[4 + i] = vc.stride(i);
  check(tops_window_attn_store(dt, B, kc.size(1), H, D, ptr(k), ptr(v), st, static_cast<const int32_t*>(ptr(n)),
                               out_ptr(kc), out_ptr(vc), ct, stream_of(k)),
        "tops_window_attn_store");
  Py_RETURN_NONE;
}

// ---------------------------------------------------------------------------
// gated norms
// ---------------------------------------------------------------------------
// Rows with contiguous channels and one stride (a copy where the tensor has no such view).
struct Rows {
  Tensor t;
  int64_t stride = 0;
  Rows(const Tensor& t0, int64_t C) : t(t0) {
    if (!t.defined()) return;
    stride = C;
    if (t.is_contiguous()) return;
    if (t.stride(-1) == 1 || C == 1) {
      // one stride for all rows: each place's is that of the next times its size
      int64_t step = -1, span = 0;
      bool uniform = true;
      for (int64_t d = t.dim() - 2; d >= 0; --d) {
        if (t.size(d) == 1) continue;
        if (step < 0)
          step = t.stride(d);
        else
          uniform = uniform && t.stride(d) == span;
        span = t.stride(d) * t.size(d);
      }
      if (uniform) {
        stride = step < 0 ? C : step;
        return;
      }
    }
    t = t.contiguous();
  }
  const void* p() const { return ptr(t); }
};

struct Norm {
  int dt, w_dt;
  int64_t C, rows, groups;
  int layer;
  Tensor w[5];  // post weight and bias, residual scale, pre weight and bias
  Norm(const Tensor& x, const Tensor& y, const Tensor& gate, PyObject* const* weights, PyObject* kind) {
    const char* k = PyUnicode_Check(kind) ? PyUnicode_AsUTF8(kind) : "";
    if (k == nullptr) throw Refused();
    layer = std::string_view(k) == "layer";
    if (!layer && std::string_view(k) != "rms")
      refuse(PyExc_ValueError, std::string("kind must be 'layer' or 'rms', got '") + k + "'");
    dt = dtype_code(x);
    must(x.dim() >= 1 && x.sizes() == y.sizes(), "x and y must have one shape (..., C)");
    C = x.size(-1);
    must(C > 0 && C <= 8192, "C must be in 1..8192");
    same_dtype(x, y, "x, y and gate");
    same_dtype(x, gate, "x, y and gate");
    rows = groups = x.numel() / C;
    must(y.device() == x.device() && (!gate.defined() || gate.device() == x.device()),
         "x, y and gate must be on one device");
    if (gate.defined() && gate.sizes() != x.sizes()) {
      const char* text = "gate must be like x, or with 1 in its last places before C";
      must(gate.dim() == x.dim() && gate.size(-1) == C, text);
      int64_t lead = x.dim() - 1;
      while (lead > 0 && gate.size(lead - 1) == 1) --lead;
      groups = 1;
      for (int64_t d = 0; d < lead; ++d) {
        must(gate.size(d) == x.size(d), text);
        groups *= gate.size(d);
      }
    }
    w_dt = -1;
    at::ScalarType first = x.scalar_type();
    for (int i = 0; i < 5; ++i) {
      w[i] = maybe(weights[i]);
      if (!w[i].defined()) continue;
      must(w[i].dim() == 1 && w[i].size(0) == C && w[i].device() == x.device(),
           "a weight must be (C,) on the device of x");
      const at::ScalarType t = w[i].scalar_type();
      if (w_dt < 0) first = t;
      if (t != first || (t != x.scalar_type() && t != at::kFloat))
        refuse(PyExc_ValueError, std::string("the weights must all be ") + at::toString(x.scalar_type()) +
                                     " or all fp32, got " + at::toString(first) + " and " + at::toString(t));
      w_dt = t == x.scalar_type() ? dt : TOPS_F32;
      w[i] = w[i].contiguous();
    }
    if (w_dt < 0) w_dt = dt;
  }
};

// (x, y, gate, 5 weights, kind, post, pre, eps) -> (h, n, stats)
PyObject* gated_norm_forward(PyObject* const* a) {
  const Tensor x = tensor(a[0]), y = tensor(a[1]), gate = maybe(a[2]);
  const Norm s(x, y, gate, a + 3, a[8]);
  const int post = flag(a[9]), pre = flag(a[10]);
  require_cuda(x);
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor h = like(x), n = pre ? like(x) : Tensor();
  at::DimVector shape(x.sizes().begin(), x.sizes().end());
  shape.back() = 4;
  const Tensor stats = empty(shape, at::kFloat, x.device());
  if (s.rows > 0) {
    const Rows rx(x, s.C), ry(y, s.C), rg(gate, s.C);
    check(tops_gated_norm_forward(s.dt, s.w_dt, s.rows, s.groups, s.C, s.layer, post, pre, static_cast<float>(real(a[11])),
                                  rx.p(), rx.stride, ry.p(), ry.stride, rg.p(), rg.stride, ptr(s.w[0]), ptr(s.w[1]),
                                  ptr(s.w[2]), ptr(s.w[3]), ptr(s.w[4]), out_ptr(h), out_ptr(n),
                                  static_cast<float*>(out_ptr(stats)), stream_of(x)),
          "tops_gated_norm_forward");
  }
  return give_tuple(h, n, stats);
}

// (dh, dn, x, y, gate, stats, 5 weights, kind, post, pre) -> (dx, dy, dgate, 5 weights')
PyObject* gated_norm_backward(PyObject* const* a) {
  const Tensor dh = maybe(a[0]), dn = maybe(a[1]), x = tensor(a[2]), y = tensor(a[3]), gate = maybe(a[4]),
               stats = tensor(a[5]);
  const Norm s(x, y, gate, a + 6, a[11]);
  const int post = flag(a[12]), pre = flag(a[13]);
  for (const Tensor* d : {&dh, &dn})
    if (d->defined()) {
      must(d->sizes() == x.sizes() && d->device() == x.device(), "dh and dn must be like x");
      same_dtype(x, *d, "x, dh and dn");
    }
  must(stats.dim() == x.dim() && stats.size(-1) == 4 && stats.sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1) &&
           stats.scalar_type() == at::kFloat && stats.is_contiguous() && stats.device() == x.device(),
       "stats must be what forward returned");
  require_cuda(x);
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor dx = like(x), dy = like(x), dgate = gate.defined() ? like(gate) : Tensor();
  Tensor dw[5];
  for (int i = 0; i < 5; ++i)
    if (s.w[i].defined()) dw[i] = like(s.w[i]);
  if (s.rows == 0) {
    if (dgate.defined()) dgate.zero_();
    for (Tensor& t : dw)
      if (t.defined()) t.zero_();
  } else {
    int64_t need = 0;
    check(tops_gated_norm_backward_workspace_bytes(s.rows, s.groups, s.C, &need), "tops_gated_norm_backward");
    const Tensor ws = empty({need}, at::kByte, x.device());
    const Rows rdh(dh, s.C), rdn(dn, s.C), rx(x, s.C), ry(y, s.C), rg(gate, s.C);
    check(tops_gated_norm_backward(s.dt, s.w_dt, s.rows, s.groups, s.C, s.layer, post, pre, rdh.p(), rdh.stride, rdn.p(),
                                   rdn.stride, rx.p(), rx.stride, ry.p(), ry.stride, rg.p(), rg.stride,
                                   static_cast<const float*>(ptr(stats)), ptr(s.w[0]), ptr(s.w[1]), ptr(s.w[2]),
                                   ptr(s.w[3]), out_ptr(dx), out_ptr(dy), out_ptr(dgate), out_ptr(dw[0]), out_ptr(dw[1]),
                                   out_ptr(dw[2]), out_ptr(dw[3]), out_ptr(dw[4]), out_ptr(ws), stream_of(x)),
          "tops_gated_norm_backward");
  }
  return give_tuple(dx, dy, dgate, dw[0], dw[1], dw[2], dw[3], dw[4]);
}

// ---------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------
// (q, k, positions, inv_freq, axis, interleaved, negate) -> (q, k)
PyObject* rotary(PyObject* const* a) {
  Tensor q = tensor(a[0]), k = maybe(a[1]);
  const Tensor pos = tensor(a[2]);
  Tensor freq = tensor(a[3]), axis = tensor(a[4]);
  const int dt = dtype_code(q), interleaved = flag(a[5]), negate = flag(a[6]);
  must(q.dim() == 4, "q must be (B, N, H, D)");
  const int64_t B = q.size(0), N = q.size(1), Hq = q.size(2), D = q.size(3);
  must(freq.dim() == 1 && freq.size(0) > 0 && 2 * freq.size(0) <= D, "inv_freq must be (P,) with 0 < 2P <= D");
  must(axis.sizes() == freq.sizes(), "axis must be (P,) like inv_freq");
  must(pos.dim() == 3 && pos.size(0) > 0 && pos.size(1) == B && pos.size(2) == N, "positions must be (axes, B, N)");
  if (freq.scalar_type() != at::kFloat || axis.scalar_type() != at::kInt)
    refuse(PyExc_ValueError, std::string("inv_freq must be fp32 and axis int32, got ") + at::toString(freq.scalar_type()) +
                                 " and " + at::toString(axis.scalar_type()));
  const bool wide = pos.scalar_type() == at::kLong;
  if (!wide && pos.scalar_type() != at::kInt)
    refuse(PyExc_ValueError, std::string("positions must be int32 or int64, got ") + at::toString(pos.scalar_type()));
  int64_t Hk = 0;
  if (k.defined()) {
    must(k.dim() == 4 && k.size(0) == B && k.size(1) == N && k.size(3) == D, "k must be (B, N, Hk, D) like q");
    same_dtype(q, k, "q and k");
    Hk = k.size(2);
  }
  must(pos.device() == q.device() && freq.device() == q.device() && axis.device() == q.device() &&
           (!k.defined() || k.device() == q.device()),
       "q, k, positions, inv_freq and axis must be on one device");
  require_cuda(q);
  const c10::cuda::CUDAGuard guard(q.device());
  const Tensor qo = like(q), ko = k.defined() ? like(k) : Tensor();
  if (q.stride(3) != 1) q = q.contiguous();
  if (k.defined() && k.stride(3) != 1) k = k.contiguous();
  freq = freq.contiguous(), axis = axis.contiguous();
  int64_t st[6] = {q.stride(0), q.stride(1), q.stride(2), 0, 0, 0};
  if (k.defined())
    for (int i = 0; i < 3; ++i) st[3 + i] = k.stride(i);
  const int64_t ps[3] = {pos.stride(0), pos.stride(1), pos.stride(2)};
  check(tops_rotary(dt, B, N, Hq, Hk, D, freq.size(0), pos.size(0), interleaved, negate, ptr(q), ptr(k), st, ptr(pos),
                    wide, ps, static_cast<const float*>(ptr(freq)), static_cast<const int32_t*>(ptr(axis)), out_ptr(qo),
                    out_ptr(ko), stream_of(q)),
        "tops_rotary");
  return give_tuple(qo, ko);
}

// ---------------------------------------------------------------------------
// the module
// ---------------------------------------------------------------------------
template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

#define TOPS_METHOD(f, n) \
  { #f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(call<f, n>)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {TOPS_METHOD(window_attn_forward, 9), TOPS_METHOD(window_attn_backward, 11),
                         TOPS_METHOD(window_attn_decode, 7),  TOPS_METHOD(window_attn_store, 5),
                         TOPS_METHOD(gated_norm_forward, 12), TOPS_METHOD(gated_norm_backward, 14),
                         TOPS_METHOD(rotary, 7),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", "Launchers of the token block's operators.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__bind() { return PyModule_Create(&module); }
