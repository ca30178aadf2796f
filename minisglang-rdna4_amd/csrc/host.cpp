// The operators' host path for plain calls, as a CPython extension: checks of shapes and types,
// outputs and workspaces from torch's caching allocator, and the C ABI call, without the interpreter
// in between. quant/kernels.py, quant/kv4.py, quant/lora.py, layers/norm.py, layers/attention.py and layers/rotary.py try it first; anything
// it does not take as it stands (op-layout weights, strided or CPU tensors, tensor subclasses, invalid
// arguments) returns None before anything is allocated or launched, and the Python path serves or
// refuses it as it always did.
//
// A decode call is bound by the host: K=N=4096 M=1 in int4 takes 5.4 us on the GPU, and took 14 us per
// call when every shape check, allocation and ctypes argument was a Python step.
//
// Nothing is kept between calls. The GIL is released around the C ABI calls (a launch may wait for
// room in its queue), as ctypes does.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdlib.h>
#include <string.h>

#include <algorithm>
#include <exception>
#include <vector>

#include "../../include/w4a8_mi355x.h"

namespace {

constexpr int kBF16 = 0, kF16 = 1, kF32 = 2;
constexpr int kScaleF16 = 0, kScaleE8M0 = 1, kScaleE4M3 = 2;
constexpr int kDecode = 1, kPrefill = 2;
constexpr int kUnsupported = 2;  // the C ABI's status for a call it leaves to another path

// the C ABI entry points, handed over once by address (they live in the library that ctypes loaded)
struct Abi {
  decltype(&w4a8_last_error) last_error;
  decltype(&w4a8_linear) linear;
  decltype(&w4a8_linear_workspace_bytes_for) linear_ws;
  decltype(&w4a8_gemm) gemm;
  decltype(&w4a8_gemm_workspace_bytes) gemm_ws;
  decltype(&w4a8_rms_norm) rms_norm;
  decltype(&w4a8_moe_padded_capacity) moe_capacity;
  decltype(&w4a8_moe_route_gemm1) moe_route_gemm1;
  decltype(&w4a8_moe_route_slots) moe_route_slots;
  decltype(&w4a8_moe_route_align) moe_route_align;
  decltype(&w4a8_moe_gemm_workspace_bytes) moe_gemm_ws;
  decltype(&w4a8_moe_gemm) moe_gemm;
  decltype(&w4a8_moe_gemm2_combine_supported) moe_g2c_supported;
  decltype(&w4a8_moe_gemm2_combine) moe_g2c;
  decltype(&w4a8_moe_gemm_quant_workspace_bytes) moe_quant_ws;
  decltype(&w4a8_moe_gemm_quant) moe_quant;
  decltype(&w4a8_moe_combine) moe_combine;
  decltype(&w4a8_kv4_append) kv4_append;
  decltype(&w4a8_kv4_read) kv4_read;
  decltype(&w4a8_kv4_attention_workspace_bytes) kv4_attention_ws;
  decltype(&w4a8_kv4_attention) kv4_attention;
  decltype(&w4a8_lora_workspace_bytes) lora_ws;
  decltype(&w4a8_lora_add) lora_add;
  decltype(&w4a8_kv4_tree) kv4_tree;
  decltype(&w4a8_kv4_tree_attention_workspace_bytes) kv4_tree_attention_ws;
  decltype(&w4a8_kv4_tree_attention) kv4_tree_attention;
  decltype(&w4a8_kv4_copy_pages) kv4_copy_pages;
  decltype(&w4a8_kv4_keep) kv4_keep;
  decltype(&w4a8_prompt_attention) prompt_attention;
  decltype(&w4a8_rotary) rotary;
};
Abi abi;
bool bound = false;

// A plain tensor argument on the GPU (torch.Tensor itself or a Parameter), or null
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous() ? &t : nullptr;
}
// an optional tensor: false when it is given and not plain
bool optional(PyObject* o, const at::Tensor*& t) {
  t = nullptr;
  if (o == Py_None) return true;
  t = plain(o);
  return t != nullptr;
}

int act_dtype(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? kBF16 : t.scalar_type() == at::kHalf ? kF16 : -1;
}
int any_dtype(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? kF32 : act_dtype(t); }

// every tensor on x's device, which is the current one
template <typename... T>
bool same_device(const at::Tensor& x, const T*... t) {
  const auto d = x.get_device();
  return d == c10::hip::current_device() && (... && (!t || t->get_device() == d));
}

// scale format of (scales, zeros) for a weight with `n` channels, `g` groups and `lead` experts (0:
// dense), or -1 when the pair is not one that the operators take as it stands
int scale_format(const at::Tensor& s, const at::Tensor* z, bool e2m1, int64_t lead, int64_t g, int64_t n) {
  const int o = lead ? 1 : 0;
  auto dims = [&](const at::Tensor& t, int64_t a, int64_t b) {
    return t.dim() == 2 + o && (!o || t.size(0) == lead) && t.size(o) == a && t.size(o + 1) == b;
  };
  if (!dims(s, g, n)) return -1;
  const auto st = s.scalar_type();
  if (st == at::kHalf) {
    if (!z) return kScaleF16;
    return !e2m1 && z->scalar_type() == at::kInt && dims(*z, g, n / 8) ? kScaleF16 : -1;
  }
  if (!e2m1) return -1;
  if (st == at::kByte && !z) return kScaleE8M0;
  if (st != at::kByte && st != at::kFloat8_e4m3fn) return -1;
  // NVFP4: the per-channel global as its int32 bits (dense: or as f32)
  if (!z || z->dim() != 1 + o || (o && z->size(0) != lead) || z->size(o) != n) return -1;
  return z->scalar_type() == at::kInt || (!o && z->scalar_type() == at::kFloat) ? kScaleE4M3 : -1;
}

at::Tensor empty(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType t) {
  return at::empty(sizes, like.options().dtype(t));
}

void* stream_of(const at::Tensor& x) { return c10::hip::getCurrentHIPStream(x.get_device()).stream(); }

PyObject* failed(int rc, const char* what) {
  const char* m = abi.last_error();
  if (m && *m) PyErr_Format(PyExc_RuntimeError, "%s: %s", what, m);
  else PyErr_Format(PyExc_RuntimeError, "%s: status %d", what, rc);
  return nullptr;
}

template <typename F>
int unlocked(F f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f();
  Py_END_ALLOW_THREADS
  return rc;
}

// C++ exceptions (an allocator out of memory) as torch's own bindings report them
template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());
  }
  return nullptr;
}

// a dense call's operands: x, w, scales, zeros, group, e2m1, x_fp8, act_scales
struct Dense {
  const at::Tensor *x, *w, *s, *z, *xq, *xs;
  int64_t M, N, K, group, wsb;
  int dt, sfmt, wfmt, arm;
  bool silu;

  int launch(void* out, int out_dt, int64_t ldo, void* ws, void* st) const {
    const int32_t* zp = z ? static_cast<const int32_t*>(z->data_ptr()) : nullptr;
    return xq ? abi.gemm(static_cast<const uint8_t*>(xq->data_ptr()), K, static_cast<const float*>(xs->data_ptr()), M,
                         w->data_ptr(), N, K, s->data_ptr(), sfmt, zp, wfmt, group, out, out_dt, ldo, silu, ws,
                         wsb > 0 ? wsb : 0, arm, st)
              : abi.linear(x->data_ptr(), dt, M, K, K, w->data_ptr(), N, s->data_ptr(), sfmt, zp, wfmt, group, out, out_dt,
                           ldo, silu, ws, wsb, arm, st);
  }
};
// false (with a Python error set, or none) when they are not what the operators take as they stand
bool dense(PyObject* const* a, bool silu, PyObject* arm, Dense& d) {
  d.x = plain(a[0]); d.w = plain(a[1]); d.s = plain(a[2]);
  if (!d.x || !d.w || !d.s || !optional(a[3], d.z) || !optional(a[6], d.xq) || !optional(a[7], d.xs) || !d.xq != !d.xs)
    return false;
  if (!PyLong_Check(a[4])) return false;
  d.group = PyLong_AsLongLong(a[4]);
  const bool e2m1 = PyObject_IsTrue(a[5]) == 1;
  d.silu = silu;
  d.arm = (int)PyLong_AsLong(arm);
  if (PyErr_Occurred()) return false;
  d.dt = act_dtype(*d.x);
  if (d.x->dim() != 2 || d.dt < 0 || d.w->scalar_type() != at::kByte || d.w->dim() != 3 || d.w->size(2) != 1024) return false;
  d.M = d.x->size(0); d.K = d.x->size(1); d.N = d.w->size(0) * 16;
  if (d.M <= 0 || d.K <= 0 || d.w->size(1) != (d.K + 127) / 128 || d.group <= 0 || d.K % d.group) return false;
  if (d.z && d.z->numel() == 0) d.z = nullptr;
  if (silu && d.N % 32) return false;
  d.sfmt = scale_format(*d.s, d.z, e2m1, 0, d.K / d.group, d.N);
  if (d.sfmt < 0 || !same_device(*d.x, d.w, d.s, d.z, d.xq, d.xs)) return false;
  if (d.xq && ((d.xq->scalar_type() != at::kByte && d.xq->scalar_type() != at::kFloat8_e4m3fn) || d.xq->dim() != 2 ||
               d.xq->size(0) != d.M || d.xq->size(1) != d.K || d.xs->scalar_type() != at::kFloat || d.xs->dim() != 1 ||
               d.xs->size(0) != d.M))
    return false;
  if (d.arm == 0) {
    const char* f = getenv("MINISGL_FORCE_TILED_LINEARS");
    d.arm = !(f && !strcmp(f, "1")) && d.M <= 16 && d.K % 32 == 0 ? kDecode : kPrefill;
  }
  d.wfmt = e2m1 ? 1 : 0;
  d.wsb = d.xq ? abi.gemm_ws(d.M, d.N, d.K, d.arm)
               : abi.linear_ws(d.M, d.N, d.K, d.sfmt, d.z != nullptr, d.wfmt, d.group, silu, d.arm);
  return true;
}

// linear(x, w, scales, zeros, group, e2m1, x_fp8, act_scales, silu, arm) -> (out, arm) or None.
// arm 0: the decode kernels for up to 16 rows of a K that is a multiple of 32, else the tiled ones, which
// MINISGL_FORCE_TILED_LINEARS=1 takes always.
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 10 || !bound) {
    PyErr_SetString(PyExc_TypeError, "linear: 10 arguments, after bind()");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    Dense d;
    const bool silu = PyObject_IsTrue(a[8]) == 1;
    if (!dense(a, silu, a[9], d)) {
      if (PyErr_Occurred()) return nullptr;
      Py_RETURN_NONE;
    }
    const int64_t nout = silu ? d.N / 2 : d.N;
    at::Tensor out = empty(*d.x, {d.M, nout}, d.x->scalar_type());
    at::Tensor ws;
    if (d.wsb > 0) ws = empty(*d.x, {d.wsb}, at::kByte);
    void* wp = ws.defined() ? ws.data_ptr() : nullptr;
    void* st = stream_of(*d.x);
    const int rc = unlocked([&] { return d.launch(out.data_ptr(), d.dt, nout, wp, st); });
    if (rc) return failed(rc, silu ? "w4a8_linear_silu" : "w4a8_linear");
    return Py_BuildValue("(Ni)", THPVariable_Wrap(std::move(out)), d.arm);
  });
}

// rms_norm(x, weight, eps, plus_one, residual, quant) -> out, (out, x_fp8, act_scales) or None
PyObject* rms_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6 || !bound) {
    PyErr_SetString(PyExc_TypeError, "rms_norm: 6 arguments, after bind()");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    const at::Tensor *x = plain(a[0]), *w, *r;
    if (!x || !optional(a[1], w) || !optional(a[4], r)) Py_RETURN_NONE;
    const double eps = PyFloat_AsDouble(a[2]);
    const bool plus_one = PyObject_IsTrue(a[3]) == 1, quant = PyObject_IsTrue(a[5]) == 1;
    if (PyErr_Occurred()) return nullptr;
    const int dt = act_dtype(*x);
    if (dt < 0 || x->dim() < 1 || x->numel() == 0) Py_RETURN_NONE;
    const int64_t K = x->size(-1), M = x->numel() / K;
    if ((w && (w->scalar_type() != x->scalar_type() || w->numel() != K)) ||
        (r && (r->scalar_type() != x->scalar_type() || r->sizes() != x->sizes())) || !same_device(*x, w, r))
      Py_RETURN_NONE;
    at::Tensor out = empty(*x, x->sizes(), x->scalar_type()), q, s;
    if (quant) {
      q = empty(*x, x->sizes(), at::kByte);
      s = empty(*x, {M}, at::kFloat);
    }
    void* st = stream_of(*x);
    const int rc = unlocked([&] {
      return abi.rms_norm(x->data_ptr(), dt, M, K, K, r ? r->data_ptr() : nullptr, K, w ? w->data_ptr() : nullptr,
                          plus_one, (float)eps, out.data_ptr(), K, quant ? static_cast<uint8_t*>(q.data_ptr()) : nullptr, K,
                          quant ? static_cast<float*>(s.data_ptr()) : nullptr, st);
    });
    if (rc) return failed(rc, "rms_norm");
    if (!quant) return THPVariable_Wrap(std::move(out));
    return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(q)),
                         THPVariable_Wrap(std::move(s)));
  });
}

struct Experts {
  const at::Tensor *w, *s, *z;
  int64_t N, K, group;
  int fmt;
};
// one expert weight (E, N/16, K tiles, 1024) with its scales; false when it is not a plain one
bool experts(PyObject* w, PyObject* s, PyObject* z, bool e2m1, int64_t E, int64_t K, Experts& e) {
  e.w = plain(w);
  e.s = plain(s);
  if (!e.w || !e.s || !optional(z, e.z)) return false;
  if (e.w->scalar_type() != at::kByte || e.w->dim() != 4 || e.w->size(3) != 1024 || e.w->size(0) != E ||
      e.w->size(2) != (K + 127) / 128 || e.s->dim() != 3 || e.s->size(1) <= 0 || K % e.s->size(1))
    return false;
  e.N = e.w->size(1) * 16;
  e.K = K;
  e.group = K / e.s->size(1);
  e.fmt = scale_format(*e.s, e.z, e2m1, E, e.s->size(1), e.N);
  return e.fmt >= 0;
}

// moe(x, w13, s13, z13, w2, s2, z2, gating, top_k, renormalize, e2m1, block_m, slots, routed, g2fuse, g2c)
// -> (out, took) or None: the silu forward of quant/kernels.py `_moe_forward` with the route computed
// here. slots: one block per slot; routed / g2fuse / g2c: the module's switches (g2c already bounded by
// the token count). took: 1 route + gemm1 in one launch, 2 gemm2 + combine in one launch.
PyObject* moe(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 16 || !bound) {
    PyErr_SetString(PyExc_TypeError, "moe: 16 arguments, after bind()");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    const at::Tensor *x = plain(a[0]), *gate = plain(a[7]);
    if (!x || !gate || x->dim() != 2 || gate->dim() != 2) Py_RETURN_NONE;
    const long top_k = PyLong_AsLong(a[8]), bm = PyLong_AsLong(a[11]);
    const bool renorm = PyObject_IsTrue(a[9]) == 1, e2m1 = PyObject_IsTrue(a[10]) == 1;
    bool slots = PyObject_IsTrue(a[12]) == 1;
    const bool routed = PyObject_IsTrue(a[13]) == 1, g2fuse = PyObject_IsTrue(a[14]) == 1, g2c = PyObject_IsTrue(a[15]) == 1;
    if (PyErr_Occurred()) return nullptr;
    const int64_t T = x->size(0), K = x->size(1), E = gate->size(1);
    const int dt = act_dtype(*x), gdt = any_dtype(*gate);
    if (dt < 0 || gdt < 0 || T <= 0 || K <= 0 || gate->size(0) != T || top_k <= 0 || top_k > E || bm <= 0) Py_RETURN_NONE;
    Experts e1, e2;
    if (!experts(a[1], a[2], a[3], e2m1, E, K, e1) || e1.N % 32) Py_RETURN_NONE;
    if (e1.group != 16 && e1.group != 32 && e1.group != 64 && e1.group != 128) Py_RETURN_NONE;
    const int64_t I = e1.N / 2;
    if (!experts(a[4], a[5], a[6], e2m1, E, I, e2) || e2.N != K) Py_RETURN_NONE;
    if (!same_device(*x, gate, e1.w, e1.s, e1.z, e2.w, e2.s, e2.z)) Py_RETURN_NONE;

    const int arm = bm < 64 ? kDecode : kPrefill, wfmt = e2m1 ? 1 : 0;
    const int64_t numel = T * top_k, P = abi.moe_capacity(numel, E, (int)bm);
    // rows enter the combine unrounded where the reference runs its fused decode gemm2 + gather-reduce
    const bool round_y2 = !(g2fuse && e2.fmt != kScaleE4M3 && e1.fmt != kScaleE4M3 && T <= 32 && bm != 128);
    const int row_dt = round_y2 ? dt : kF32;
    const bool fuse2 = g2fuse && g2c && arm == kDecode &&
                       abi.moe_g2c_supported(I, e2.fmt, e2.z != nullptr, wfmt, e2.group, (int)top_k) == 1;
    const int64_t ws1 = abi.moe_gemm_ws(numel, E, (int)bm, P, e1.N, K, arm);
    const int64_t ws2 = fuse2 ? 0 : abi.moe_quant_ws(P, I);
    // every intermediate in one allocation, each 256-byte aligned
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
      const int64_t o = at;
      at += (bytes + 255) / 256 * 256;
      return o;
    };
    const int64_t o_tw = take(numel * 4), o_ids = take(numel * 4), o_sorted = take(P * 4),
                  o_eid = take((P + bm - 1) / bm * 4), o_ntp = take(4), o_inv = take(numel * 4), o_xq = take(T * K),
                  o_xs = take(T * 4), o_b2 = take(P * I * 2), o_ws1 = take(ws1 > 0 ? ws1 : 0),
                  o_ws2 = take(ws2 > 0 ? ws2 : 0), o_y2 = take(fuse2 ? 0 : P * K * (row_dt == kF32 ? 4 : 2));
    at::Tensor out = empty(*x, {T, K}, x->scalar_type()), mem = empty(*x, {at}, at::kByte);
    uint8_t* m = static_cast<uint8_t*>(mem.data_ptr());
    auto f32 = [&](int64_t o) { return reinterpret_cast<float*>(m + o); };
    auto i32 = [&](int64_t o) { return reinterpret_cast<int32_t*>(m + o); };
    auto zp = [](const Experts& e) { return e.z ? static_cast<const int32_t*>(e.z->data_ptr()) : nullptr; };
    void* st = stream_of(*x);
    int took = 0;
    const char* what = "";
    const int rc = unlocked([&]() -> int {
      int r = kUnsupported;
      if (slots && routed && numel <= E && numel * bm <= P) {
        what = "w4a8_moe route_gemm1";
        r = abi.moe_route_gemm1(gate->data_ptr(), gdt, T, E, (int)top_k, renorm, x->data_ptr(), dt, K, (int)bm, P,
                                e1.w->data_ptr(), e1.N, K, e1.s->data_ptr(), e1.fmt, zp(e1), wfmt, e1.group, f32(o_tw),
                                i32(o_ids), i32(o_sorted), i32(o_eid), i32(o_ntp), i32(o_inv), m + o_b2, dt, I, st);
        if (r == 0) took |= 1;
        else if (r != kUnsupported) return r;
      }
      if (r) {
        // the grouped GEMMs size their grids for at most numel / block + min(E, numel) blocks
        const bool sl = slots && numel <= E && numel * bm <= P;
        what = sl ? "moe_route_slots" : "moe_route_align";
        r = (sl ? abi.moe_route_slots : abi.moe_route_align)(
            gate->data_ptr(), gdt, T, E, (int)top_k, renorm, (int)bm, P, f32(o_tw), i32(o_ids), i32(o_sorted),
            i32(o_eid), i32(o_ntp), i32(o_inv), x->data_ptr(), dt, K, K, m + o_xq, K, f32(o_xs), st);
        if (r) return r;
        what = "w4a8_moe gemm1";
        r = abi.moe_gemm(m + o_xq, K, f32(o_xs), 1, i32(o_sorted), i32(o_eid), i32(o_ntp), numel, (int)top_k, (int)bm, P,
                         e1.w->data_ptr(), E, e1.N, K, e1.s->data_ptr(), e1.fmt, zp(e1), wfmt, e1.group, m + o_b2, dt, I,
                         1, ws1 > 0 ? m + o_ws1 : nullptr, ws1, arm, st);
        if (r) return r;
      }
      if (fuse2) {
        took |= 2;
        what = "w4a8_moe gemm2+combine";
        return abi.moe_g2c(m + o_b2, dt, I, i32(o_ids), f32(o_tw), i32(o_inv), T, (int)top_k, (int)bm, P,
                           e2.w->data_ptr(), E, K, I, e2.s->data_ptr(), e2.fmt, zp(e2), wfmt, e2.group, out.data_ptr(), dt,
                           K, row_dt, st);
      }
      what = "w4a8_moe gemm2";
      r = abi.moe_quant(m + o_b2, dt, I, i32(o_sorted), i32(o_eid), i32(o_ntp), numel, (int)bm, P, e2.w->data_ptr(), E, K,
                        I, e2.s->data_ptr(), e2.fmt, zp(e2), wfmt, e2.group, m + o_y2, row_dt, K, m + o_ws2, ws2, arm, st);
      if (r) return r;
      what = "w4a8_moe combine";
      return abi.moe_combine(m + o_y2, row_dt, K, i32(o_inv), f32(o_tw), T, (int)top_k, K, out.data_ptr(), dt, st);
    });
    if (rc) return failed(rc, what);
    return Py_BuildValue("(Ni)", THPVariable_Wrap(std::move(out)), took);
  });
}

// ---- the 4-bit cache (quant/kv4.py) and the low-rank adapters (quant/lora.py)

// a tensor on the GPU with any strides, or null
const at::Tensor* strided(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.layout() == at::kStrided ? &t : nullptr;
}
bool aligned16(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15u) == 0; }

// (T, heads, D) rows that the kernels take as they stand
bool head_rows(const at::Tensor* t, at::ScalarType st, int64_t D) {
  return t && t->dim() == 3 && t->scalar_type() == st && t->size(2) == D && t->stride(2) == 1 &&
         (t->size(0) <= 1 || t->stride(0) % 8 == 0) && (t->size(1) <= 1 || t->stride(1) % 8 == 0) && aligned16(*t);
}
// (M, N) rows that the kernels take as they stand
bool flat_rows(const at::Tensor* t, at::ScalarType st, int64_t M, int64_t N) {
  return t && t->dim() == 2 && t->scalar_type() == st && t->size(0) == M && t->size(1) == N && t->stride(1) == 1 &&
         (M == 1 || (t->stride(0) % 8 == 0 && t->stride(0) >= N)) && aligned16(*t);
}

// the cache's tensors (k, v, k_scale, v_scale: checked by KV4Cache) and a ragged batch (page table, cu, lens)
struct Kv4 {
  const at::Tensor *k, *v, *ks, *vs, *table, *cu, *lens;
  int64_t pages, H, page, D, B, width, ldt;
  int dt;
};
bool kv4(PyObject* const* a, Kv4& c) {
  const at::Tensor** t[] = {&c.k, &c.v, &c.ks, &c.vs};
  for (int i = 0; i < 4; ++i)
    if (!(*t[i] = plain(a[i]))) return false;
  c.table = strided(a[4]);
  c.cu = plain(a[5]);
  c.lens = plain(a[6]);
  if (!c.table || !c.cu || !c.lens || c.k->dim() != 4) return false;
  c.pages = c.k->size(0); c.H = c.k->size(1); c.page = c.k->size(2); c.D = c.k->size(3) * 2;
  c.dt = act_dtype(*c.ks);
  if (c.dt < 0 || c.table->dim() != 2 || c.cu->dim() != 1 || c.lens->dim() != 1) return false;
  for (const at::Tensor* m : {c.table, c.cu, c.lens})
    if (m->scalar_type() != at::kInt) return false;
  c.B = c.lens->size(0);
  c.width = c.table->size(1);
  if (c.cu->size(0) != c.B + 1 || c.table->size(0) != c.B || c.B < 1 || (c.width > 1 && c.table->stride(1) != 1) ||
      (c.B > 1 && c.table->stride(0) < c.width))
    return false;
  c.ldt = c.B > 1 ? c.table->stride(0) : c.width;
  return true;
}
const int32_t* i32(const at::Tensor* t) { return static_cast<const int32_t*>(t->data_ptr()); }

// kv4_append(k cache, v cache, k_scale, v_scale, page_table, cu, lens, k, v) -> True or None
PyObject* kv4_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9 || !bound) {
    PyErr_SetString(PyExc_TypeError, "kv4_append: 9 arguments, after bind()");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    Kv4 c;
    if (!kv4(a, c)) Py_RETURN_NONE;
    const at::Tensor *k = strided(a[7]), *v = strided(a[8]);
    if (!head_rows(k, c.ks->scalar_type(), c.D) || !head_rows(v, c.ks->scalar_type(), c.D) || k->size(1) != c.H ||
        v->size(1) != c.H || k->size(0) != v->size(0) ||
        !same_device(*k, v, c.k, c.v, c.ks, c.vs, c.table, c.cu, c.lens))
      Py_RETURN_NONE;
    void* st = stream_of(*k);
    const int rc = unlocked([&] {
      return abi.kv4_append(k->data_ptr(), k->stride(0), k->stride(1), v->data_ptr(), v->stride(0), v->stride(1), c.dt,
                            k->size(0), c.H, c.D, c.k->data_ptr(), c.v->data_ptr(), c.ks->data_ptr(), c.vs->data_ptr(),
                            c.pages, c.page, i32(c.table), c.ldt, c.width, i32(c.cu), i32(c.lens), c.B, st);
    });
    if (rc) return failed(rc, "kv4_append");
    Py_RETURN_TRUE;
  });
}

// kv4_read(cache and batch as above, rows) -> (k, v) or None
PyObject* kv4_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8 || !bound) {
    PyErr_SetString(PyExc_TypeError, "kv4_read: 8 arguments, after bind()");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    Kv4 c;
    if (!kv4(a, c) || !PyLong_Check(a[7])) Py_RETURN_NONE;
    const int64_t T = PyLong_AsLongLong(a[7]);
    if (PyErr_Occurred()) return nullptr;
    if (T < 0 || !same_device(*c.k, c.v, c.ks, c.vs, c.table, c.cu, c.lens)) Py_RETURN_NONE;
    at::Tensor k = empty(*c.k, {T, c.H, c.D}, c.ks->scalar_type()), v = empty(*c.k, {T, c.H, c.D}, c.ks->scalar_type());
    void* st = stream_of(k);
    const int rc = unlocked([&] {
      return abi.kv4_read(c.k->data_ptr(), c.v->data_ptr(), c.ks->data_ptr(), c.vs->data_ptr(), c.dt, c.pages, c.page, c.H,
                          c.D, i32(c.table), c.ldt, c.width, i32(c.cu), i32(c.lens), c.B, T, k.data_ptr(), v.data_ptr(), st);
    });
    if (rc) return failed(rc, "kv4_read");
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(k)), THPVariable_Wrap(std::move(v)));
  });
}

// attention over the cache: q = a[7], max_q = a[8], max_kv = a[9], scale = a[10], then causal (null: a tree, with its
// mask and positions), window, out and lse
PyObject* attend(PyObject* const* a, PyObject* pcausal, PyObject* pwindow, PyObject* pout, PyObject* plse, PyObject* pmask,
                 PyObject* ppos) {
  Kv4 c;
  if (!kv4(a, c)) Py_RETURN_NONE;
  const at::Tensor *q = strided(a[7]), *o = pout == Py_None ? nullptr : strided(pout), *mask = nullptr, *pos = nullptr;
  if (!head_rows(q, c.ks->scalar_type(), c.D) || (pout != Py_None && !head_rows(o, q->scalar_type(), c.D)))
    Py_RETURN_NONE;
  const int64_t T = q->size(0), Hq = q->size(1);
  if (pmask) {
    mask = plain(pmask);
    pos = plain(ppos);
    if (!mask || !pos || mask->scalar_type() != at::kInt || pos->scalar_type() != at::kInt || mask->dim() != 2 ||
        pos->dim() != 1 || mask->size(0) != T || pos->size(0) != T || mask->size(1) < 1 || mask->size(1) > 128)
      Py_RETURN_NONE;
  }
  if ((o && (o->size(0) != T || o->size(1) != Hq)) ||
      !same_device(*q, o, c.k, c.v, c.ks, c.vs, c.table, c.cu, c.lens, mask, pos) || Hq < c.H || Hq % c.H)
    Py_RETURN_NONE;
  const int64_t cap = c.width * c.page;
  int64_t max_q = T, max_kv = cap;
  if ((a[8] != Py_None && !PyLong_Check(a[8])) || (a[9] != Py_None && !PyLong_Check(a[9])) || !PyLong_Check(pwindow))
    Py_RETURN_NONE;
  if (a[8] != Py_None) max_q = std::min<int64_t>(PyLong_AsLongLong(a[8]), T);
  if (a[9] != Py_None) max_kv = std::min<int64_t>(PyLong_AsLongLong(a[9]), cap);
  const double scale = PyFloat_AsDouble(a[10]);
  const int64_t window = PyLong_AsLongLong(pwindow);
  const bool causal = !pcausal || PyObject_IsTrue(pcausal) == 1, want_lse = PyObject_IsTrue(plse) == 1;
  if (PyErr_Occurred()) return nullptr;
  if (window < 0 || max_q < 0 || max_kv < 0) Py_RETURN_NONE;
  if (window) max_kv = std::min(max_kv, window + max_q);
  const int64_t wsb = mask ? abi.kv4_tree_attention_ws(T, Hq, c.H, c.D, c.B, window, max_q, max_kv)
                           : abi.kv4_attention_ws(T, Hq, c.H, c.D, c.B, max_q, max_kv);
  at::Tensor out = o ? *o : empty(*q, {T, Hq, c.D}, q->scalar_type()), lse, ws;
  if (want_lse) lse = empty(*q, {T, Hq}, at::kFloat);
  if (wsb > 0) ws = empty(*q, {wsb}, at::kByte);
  void* st = stream_of(*q);
  float* lp = want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr;
  void* wp = ws.defined() ? ws.data_ptr() : nullptr;
  const int rc = unlocked([&] {
    if (mask)
      return abi.kv4_tree_attention(q->data_ptr(), c.dt, q->stride(0), q->stride(1), T, Hq, c.H, c.D, c.k->data_ptr(),
                                    c.v->data_ptr(), c.ks->data_ptr(), c.vs->data_ptr(), c.pages, c.page, i32(c.table), c.ldt,
                                    c.width, i32(c.cu), i32(c.lens), c.B, (float)scale, window, max_q, max_kv,
                                    reinterpret_cast<const uint32_t*>(i32(mask)), mask->size(1), mask->size(1), i32(pos),
                                    out.data_ptr(), out.stride(0), out.stride(1), lp, wp, wsb > 0 ? wsb : 0, st);
    return abi.kv4_attention(q->data_ptr(), c.dt, q->stride(0), q->stride(1), T, Hq, c.H, c.D, c.k->data_ptr(),
                             c.v->data_ptr(), c.ks->data_ptr(), c.vs->data_ptr(), c.pages, c.page, i32(c.table), c.ldt,
                             c.width, i32(c.cu), i32(c.lens), c.B, (float)scale, causal, window, max_q, max_kv,
                             out.data_ptr(), out.stride(0), out.stride(1), lp, wp, wsb > 0 ? wsb : 0, st);
  });
  if (rc) return failed(rc, "kv4_attention");
  PyObject* po = o ? Py_NewRef(pout) : THPVariable_Wrap(std::move(out));
  PyObject* pl = want_lse ? THPVariable_Wrap(std::move(lse)) : Py_NewRef(Py_None);
  return Py_BuildValue("(NN)", po, pl);
}

// kv4_attention(cache and batch, q, max_q or None, max_kv or None, scale, causal, window, out or None, lse)
// -> (out, lse or None) or None
PyObject* kv4_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 15 || !bound) {
    PyErr_SetString(PyExc_TypeError, "kv4_attention: 15 arguments, after bind()");
    return nullptr;
  }
  return guarded([&]() -> PyObject* { return attend(a, a[11], a[12], a[13], a[14], nullptr, nullptr); });
}

// kv4_tree_attention(cache and batch, q, max_q or None, max_kv or None, scale, window, out or None, lse, mask, positions)
// -> (out, lse or None) or None
PyObject* kv4_tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 16 || !bound) {
    PyErr_SetString(PyExc_TypeError, "kv4_tree_attention: 16 arguments, after bind()");
    return nullptr;
  }
  return guarded([&]() -> PyObject* { return attend(a, nullptr, a[11], a[12], a[13], a[14], a[15]); });
}

bool ints(const at::Tensor* t, int64_t dim) { return t && t->scalar_type() == at::kInt && t->dim() == dim; }

// kv4_tree(parents, cu, lens, max_q, window) -> (mask, positions) or None
PyObject* kv4_tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 5 || !bound) {
    PyErr_SetString(PyExc_TypeError, "kv4_tree: 5 arguments, after bind()");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    const at::Tensor *parents = plain(a[0]), *cu = plain(a[1]), *lens = plain(a[2]);
    if (!ints(parents, 1) || !ints(cu, 1) || !ints(lens, 1) || !PyLong_Check(a[3]) || !PyLong_Check(a[4])) Py_RETURN_NONE;
    const int64_t max_q = PyLong_AsLongLong(a[3]), window = PyLong_AsLongLong(a[4]);
    if (PyErr_Occurred()) return nullptr;
    const int64_t T = parents->size(0), B = lens->size(0);
    if (max_q < 1 || max_q > 4096 || window < 0 || cu->size(0) != B + 1 || !same_device(*parents, cu, lens)) Py_RETURN_NONE;
    const int64_t words = (max_q + 31) / 32;
    at::Tensor mask = empty(*parents, {T, words}, at::kInt), pos = empty(*parents, {T}, at::kInt);
    void* st = stream_of(*parents);
    const int rc = unlocked([&] {
      return abi.kv4_tree(i32(parents), T, i32(cu), i32(lens), B, words, window, static_cast<uint32_t*>(mask.data_ptr()),
                          static_cast<int32_t*>(pos.data_ptr()), st);
    });
    if (rc) return failed(rc, "kv4_tree");
    return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(mask)), THPVariable_Wrap(std::move(pos)));
  });
}

// caches of one shape, as a tuple of four tensors each: their pointers, and the first one's tensors in `c`
bool caches(PyObject* o, std::vector<const void*>& arrays, const at::Tensor* (&c)[4]) {
  if (!PyTuple_CheckExact(o)) return false;
  const Py_ssize_t n = PyTuple_GET_SIZE(o);
  if (n < 4 || n % 4) return false;
  arrays.reserve(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor* t = plain(PyTuple_GET_ITEM(o, i));
    if (!t || t->dim() != 4) return false;
    if (i < 4) c[i] = t;
    if (t->scalar_type() != c[i % 4]->scalar_type() || t->sizes() != c[i % 4]->sizes() || !same_device(*c[0], t)) return false;
    if (i % 4 == 0)
      for (Py_ssize_t j = 0; j < i; j += 4)
        if (arrays[j] == t->data_ptr()) return false;
    arrays.push_back(t->data_ptr());
  }
  return true;
}

// kv4_copy_pages(caches' tensors, src, dst) -> True or None
PyObject* kv4_copy_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3 || !bound) {
    PyErr_SetString(PyExc_TypeError, "kv4_copy_pages: 3 arguments, after bind()");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    std::vector<const void*> arrays;
    const at::Tensor* c[4];
    const at::Tensor *src = plain(a[1]), *dst = plain(a[2]);
    if (!ints(src, 1) || !ints(dst, 1) || src->size(0) != dst->size(0) || !caches(a[0], arrays, c) ||
        !same_device(*c[0], src, dst))
      Py_RETURN_NONE;
    void* st = stream_of(*src);
    const int rc = unlocked([&] {
      return abi.kv4_copy_pages(arrays.data(), (int64_t)arrays.size() / 4, c[0]->size(0), c[0]->size(2), c[0]->size(1),
                                c[0]->size(3) * 2, i32(src), i32(dst), src->size(0), st);
    });
    if (rc) return failed(rc, "kv4_copy_pages");
    Py_RETURN_TRUE;
  });
}

// kv4_keep(caches' tensors, page_table, cu, lens, keep, kept) -> new lengths or None
PyObject* kv4_keep(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6 || !bound) {
    PyErr_SetString(PyExc_TypeError, "kv4_keep: 6 arguments, after bind()");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    std::vector<const void*> arrays;
    const at::Tensor* c[4];
    const at::Tensor *keep = plain(a[4]), *kept = plain(a[5]);
    if (!ints(keep, 2) || !ints(kept, 1) || !caches(a[0], arrays, c)) Py_RETURN_NONE;
    PyObject* const first[7] = {PyTuple_GET_ITEM(a[0], 0), PyTuple_GET_ITEM(a[0], 1), PyTuple_GET_ITEM(a[0], 2),
                                PyTuple_GET_ITEM(a[0], 3), a[1], a[2], a[3]};
    Kv4 s;
    if (!kv4(first, s) || keep->size(0) != s.B || kept->size(0) != s.B ||
        !same_device(*c[0], s.table, s.cu, s.lens, keep, kept))
      Py_RETURN_NONE;
    at::Tensor now = empty(*kept, {s.B}, at::kInt);
    void* st = stream_of(*kept);
    const int rc = unlocked([&] {
      return abi.kv4_keep(arrays.data(), (int64_t)arrays.size() / 4, s.pages, s.page, s.H, s.D, i32(s.table), s.ldt, s.width,
                          i32(s.cu), i32(s.lens), s.B, i32(keep), keep->size(1), keep->size(1), i32(kept),
                          static_cast<int32_t*>(now.data_ptr()), st);
    });
    if (rc) return failed(rc, "kv4_keep");
    return THPVariable_Wrap(std::move(now));
  });
}

// prompt_attention(q, k, v, cu, max_q or None, scale, causal, window, out or None, lse) -> (out, lse or None) or None
PyObject* prompt_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 10 || !bound) {
    PyErr_SetString(PyExc_TypeError, "prompt_attention: 10 arguments, after bind()");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    const at::Tensor *q = strided(a[0]), *k = strided(a[1]), *v = strided(a[2]), *cu = plain(a[3]);
    const at::Tensor* o = a[8] == Py_None ? nullptr : strided(a[8]);
    if (!q || !ints(cu, 1) || cu->size(0) < 1 || q->dim() != 3 || act_dtype(*q) < 0) Py_RETURN_NONE;
    const int64_t T = q->size(0), Hq = q->size(1), D = q->size(2);
    const auto t = q->scalar_type();
    if ((D != 64 && D != 128 && D != 256) || !head_rows(q, t, D) || !head_rows(k, t, D) || !head_rows(v, t, D) ||
        (a[8] != Py_None && !head_rows(o, t, D)))
      Py_RETURN_NONE;
    const int64_t H = k->size(1);
    for (const at::Tensor* r : {k, v})
      if (r->size(0) != T || r->size(1) != H || (T > 1 && (r->stride(0) < D || r->stride(0) >= 1 << 23))) Py_RETURN_NONE;
    if (H < 1 || Hq < H || Hq % H || (o && (o->size(0) != T || o->size(1) != Hq)) || !same_device(*q, k, v, cu, o))
      Py_RETURN_NONE;
    if ((a[4] != Py_None && !PyLong_Check(a[4])) || !PyLong_Check(a[7])) Py_RETURN_NONE;
    const int64_t max_q = a[4] == Py_None ? T : std::min<int64_t>(PyLong_AsLongLong(a[4]), T);
    const double scale = PyFloat_AsDouble(a[5]);
    const int64_t window = PyLong_AsLongLong(a[7]);
    const bool causal = PyObject_IsTrue(a[6]) == 1, want_lse = PyObject_IsTrue(a[9]) == 1;
    if (PyErr_Occurred()) return nullptr;
    if (window < 0 || max_q < 0) Py_RETURN_NONE;
    at::Tensor out = o ? *o : empty(*q, {T, Hq, D}, t), lse;
    if (want_lse) lse = empty(*q, {T, Hq}, at::kFloat);
    void* st = stream_of(*q);
    const int rc = unlocked([&] {
      return abi.prompt_attention(q->data_ptr(), q->stride(0), q->stride(1), k->data_ptr(), k->stride(0), k->stride(1),
                                  v->data_ptr(), v->stride(0), v->stride(1), act_dtype(*q), T, Hq, H, D, i32(cu),
                                  cu->size(0) - 1, (float)scale, causal, window, max_q, out.data_ptr(), out.stride(0),
                                  out.stride(1), want_lse ? static_cast<float*>(lse.data_ptr()) : nullptr, st);
    });
    if (rc) return failed(rc, "prompt_attention");
    PyObject* po = o ? Py_NewRef(a[8]) : THPVariable_Wrap(std::move(out));
    PyObject* pl = want_lse ? THPVariable_Wrap(std::move(lse)) : Py_NewRef(Py_None);
    return Py_BuildValue("(NN)", po, pl);
  });
}

// rotary(turns, axis, axes, head_dim, rotary_dim, adjacent, scale, q, k, positions, in place) -> (q, k) or None
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 11 || !bound) {
    PyErr_SetString(PyExc_TypeError, "rotary: 11 arguments, after bind()");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    const at::Tensor *turns = plain(a[0]), *axis = plain(a[1]), *q = strided(a[7]), *k = strided(a[8]), *pos = plain(a[9]);
    if (!turns || !axis || !q || !k || !pos) Py_RETURN_NONE;
    const int64_t axes = PyLong_AsLongLong(a[2]), D = PyLong_AsLongLong(a[3]), R = PyLong_AsLongLong(a[4]);
    const bool adjacent = PyObject_IsTrue(a[5]) == 1, inplace = PyObject_IsTrue(a[10]) == 1;
    const double scale = PyFloat_AsDouble(a[6]);
    if (PyErr_Occurred()) return nullptr;
    const auto t = q->scalar_type();
    if (act_dtype(*q) < 0 || !head_rows(q, t, D) || !head_rows(k, t, D)) Py_RETURN_NONE;
    const int64_t T = q->size(0), Hq = q->size(1), Hk = k->size(1);
    const bool wide = pos->scalar_type() == at::kLong;
    if (k->size(0) != T || Hq < 1 || Hk < 1 || (!wide && pos->scalar_type() != at::kInt) || turns->numel() != R / 2 ||
        axis->numel() != R / 2 || !same_device(*q, k, pos, turns, axis))
      Py_RETURN_NONE;
    if (!(pos->dim() == 2 && pos->size(0) == axes && pos->size(1) == T) && !(pos->dim() == 1 && axes == 1 && pos->size(0) == T))
      Py_RETURN_NONE;
    at::Tensor qo = inplace ? *q : empty(*q, {T, Hq, D}, t), ko = inplace ? *k : empty(*k, {T, Hk, D}, t);
    void* st = stream_of(*q);
    const int rc = unlocked([&] {
      return abi.rotary(q->data_ptr(), q->stride(0), q->stride(1), Hq, k->data_ptr(), k->stride(0), k->stride(1), Hk,
                        act_dtype(*q), T, D, R, adjacent, pos->data_ptr(), wide, axes, T,
                        static_cast<const uint64_t*>(turns->data_ptr()), i32(axis), (float)scale, qo.data_ptr(), qo.stride(0),
                        qo.stride(1), ko.data_ptr(), ko.stride(0), ko.stride(1), st);
    });
    if (rc) return failed(rc, "Rotary");
    PyObject* pq = inplace ? Py_NewRef(a[7]) : THPVariable_Wrap(std::move(qo));
    PyObject* pk = inplace ? Py_NewRef(a[8]) : THPVariable_Wrap(std::move(ko));
    return Py_BuildValue("(NN)", pq, pk);
  });
}

// the adapters (a, b, scaling: checked by LoraAdapters), the host's slice widths and the rows' adapters
struct Lora {
  const at::Tensor *a, *b, *s, *ids;
  int64_t L, N, rank, K;
  int64_t cols[16];
  int slices;
};
bool lora(PyObject* const* o, Lora& l) {
  l.a = plain(o[0]); l.b = plain(o[1]); l.s = plain(o[2]); l.ids = plain(o[4]);
  if (!l.a || !l.b || !l.s || !l.ids || l.a->dim() != 3 || l.b->dim() != 3 || !PyTuple_CheckExact(o[3])) return false;
  l.slices = (int)PyTuple_GET_SIZE(o[3]);
  if (l.slices < 1 || l.slices > 16) return false;
  for (int i = 0; i < l.slices; ++i) {
    l.cols[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(o[3], i));
    if (PyErr_Occurred()) return false;
  }
  l.L = l.b->size(0); l.N = l.b->size(1); l.rank = l.b->size(2); l.K = l.a->size(2);
  return l.ids->scalar_type() == at::kInt && l.ids->dim() == 1;
}
int add_adapters(const at::Tensor& x, const Lora& l, const void* base, int base_dt, int64_t ldb, void* out, int64_t ldo,
                 void* ws, int64_t wsb, void* st) {
  const int64_t M = x.size(0);
  return abi.lora_add(x.data_ptr(), act_dtype(x), M, l.K, M > 1 ? x.stride(0) : l.K, l.a->data_ptr(), l.b->data_ptr(),
                      static_cast<const float*>(l.s->data_ptr()), l.L, l.rank, l.cols, l.slices, i32(l.ids), base, base_dt,
                      ldb, out, ldo, ws, wsb, st);
}

// lora_add(a, b, scaling, slices, adapters, y, x, out) -> True or None
PyObject* lora_add(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8 || !bound) {
    PyErr_SetString(PyExc_TypeError, "lora_add: 8 arguments, after bind()");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    Lora l;
    if (!lora(a, l)) {
      if (PyErr_Occurred()) return nullptr;
      Py_RETURN_NONE;
    }
    const at::Tensor *y = strided(a[5]), *x = strided(a[6]), *o = strided(a[7]);
    const int64_t M = l.ids->size(0);
    const auto t = l.a->scalar_type();
    if (M < 1 || !flat_rows(x, t, M, l.K) || !flat_rows(y, t, M, l.N) || !flat_rows(o, t, M, l.N) ||
        !same_device(*x, y, o, l.a, l.b, l.s, l.ids))
      Py_RETURN_NONE;
    const int64_t wsb = abi.lora_ws(M, l.K, l.rank, l.slices);
    if (wsb < 0) Py_RETURN_NONE;
    at::Tensor ws = empty(*x, {wsb}, at::kByte);
    void* st = stream_of(*x);
    const int rc = unlocked([&] {
      return add_adapters(*x, l, y->data_ptr(), act_dtype(*y), M > 1 ? y->stride(0) : l.N, o->data_ptr(),
                          M > 1 ? o->stride(0) : l.N, ws.data_ptr(), wsb, st);
    });
    if (rc) return failed(rc, "lora_add");
    Py_RETURN_TRUE;
  });
}

// linear_lora(a, b, scaling, slices, adapters, x, w, scales, zeros, group, e2m1, x_fp8, act_scales, arm)
// -> out or None: linear() above with arm 0, 1 or 2, its output in f32 until the adapters are added
PyObject* linear_lora(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 14 || !bound) {
    PyErr_SetString(PyExc_TypeError, "linear_lora: 14 arguments, after bind()");
    return nullptr;
  }
  return guarded([&]() -> PyObject* {
    Lora l;
    if (!lora(a, l)) {
      if (PyErr_Occurred()) return nullptr;
      Py_RETURN_NONE;
    }
    Dense d;
    if (!dense(a + 5, false, a[13], d)) {
      if (PyErr_Occurred()) return nullptr;
      Py_RETURN_NONE;
    }
    if (d.x->scalar_type() != l.a->scalar_type() || d.K != l.K || d.N != l.N || l.ids->size(0) != d.M || !aligned16(*d.x) ||
        !same_device(*d.x, l.a, l.b, l.s, l.ids))
      Py_RETURN_NONE;
    const int64_t lwb = abi.lora_ws(d.M, l.K, l.rank, l.slices);
    if (lwb < 0) Py_RETURN_NONE;
    // the projection's workspace, the adapters' one and the f32 output in one allocation
    const int64_t at1 = (std::max<int64_t>(d.wsb, 0) + 255) / 256 * 256, at2 = at1 + (lwb + 255) / 256 * 256;
    at::Tensor out = empty(*d.x, {d.M, d.N}, d.x->scalar_type());
    at::Tensor mem = empty(*d.x, {at2 + d.M * d.N * 4}, at::kByte);
    uint8_t* m = static_cast<uint8_t*>(mem.data_ptr());
    void* base = m + at2;
    void* st = stream_of(*d.x);
    const char* what = "w4a8_linear";
    const int rc = unlocked([&] {
      const int r = d.launch(base, kF32, d.N, m, st);
      if (r) return r;
      what = "w4a8_linear_lora";
      return add_adapters(*d.x, l, base, kF32, d.N, out.data_ptr(), d.N, m + at1, lwb, st);
    });
    if (rc) return failed(rc, what);
    return THPVariable_Wrap(std::move(out));
  });
}

// bind(address of each entry point in Abi's order)
PyObject* bind(PyObject*, PyObject* args) {
  constexpr Py_ssize_t kCount = sizeof(Abi) / sizeof(void*);
  if (PyTuple_GET_SIZE(args) != kCount) {
    PyErr_Format(PyExc_TypeError, "bind: %zd addresses", kCount);
    return nullptr;
  }
  void* p[kCount];
  for (Py_ssize_t i = 0; i < kCount; ++i) {
    p[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(args, i));
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: a null address");
      return nullptr;
    }
  }
  memcpy(&abi, p, sizeof abi);
  bound = true;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear)), METH_FASTCALL, nullptr},
    {"rms_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rms_norm)), METH_FASTCALL, nullptr},
    {"moe", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(moe)), METH_FASTCALL, nullptr},
    {"kv4_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kv4_append)), METH_FASTCALL, nullptr},
    {"kv4_read", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kv4_read)), METH_FASTCALL, nullptr},
    {"kv4_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kv4_attention)), METH_FASTCALL, nullptr},
    {"kv4_tree", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kv4_tree)), METH_FASTCALL, nullptr},
    {"kv4_tree_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kv4_tree_attention)), METH_FASTCALL,
     nullptr},
    {"kv4_copy_pages", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kv4_copy_pages)), METH_FASTCALL, nullptr},
    {"kv4_keep", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kv4_keep)), METH_FASTCALL, nullptr},
    {"prompt_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(prompt_attention)), METH_FASTCALL, nullptr},
    {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rotary)), METH_FASTCALL, nullptr},
    {"lora_add", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(lora_add)), METH_FASTCALL, nullptr},
    {"linear_lora", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(linear_lora)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "w4a8_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_w4a8_host() {
  PyObject* m = PyModule_Create(&module_def);
  if (m && PyModule_AddStringConstant(m, "built_for", W4A8_BUILT_FOR) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
