// The decode attention calls from torch tensors to the C ABI in native code.
//
// A decode layer's launch takes 5-7 us on the GPU for small batches; checking
// nine tensors, reading their strides and building a forty-argument ctypes call
// in Python took about 12 us of host time per call, so a loop over layers ran
// at the host's pace. With this path it runs at the GPU's, measured on MI355X as
// back-to-back calls: one sequence of 300 tokens 12.2 -> 5.6 us per call (head_dim
// 64, 14 / 2 heads, rotary form), 8 of up to 512 12.6 -> 6.3 (write form), 128 of
// up to 1088 12.3 -> 11.4. The calls on the 8-bit pool and of the drafts' verification take
// the same path: a decode step's write 9.4 -> 4.4 us, a document's read 11.6 -> 5.5, one
// sequence of 300 tokens 12.7 -> 5.8.
//
// Each function launches the call it is given, or returns None without having
// done anything when something about it is not plain: another device than the
// current one, a type, shape, alignment or stride the Python entry point
// refuses or copies, a tensor subclass, a functorch wrapper, an active
// __torch_function__ or dispatch mode, or a workspace too small. The Python entry
// point then runs its own checks, with its own errors, and its own call. Where the
// library reports a HIP error, the status is returned for the caller to raise: the
// call was made, or the error is an earlier one that only this report tells of.
//
// The module is not linked against the library: bind() is given the addresses
// of the library the process has loaded, whatever file that is.
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include "paged_attention.h"

namespace {

using at::Tensor;
using Obj = py::handle;

#define PA_HOST_CALLS(X)                    \
  X(pa_decode_batched_workspace_bytes)      \
  X(pa_decode_rope_batched_workspace_bytes) \
  X(pa_decode_batched_f16)                  \
  X(pa_decode_kv_write_batched_f16)         \
  X(pa_decode_rope_batched_f16)

// Those of the 8-bit pool and of the drafts' verification, bound apart (bind_fp8).
#define PA_HOST_CALLS_FP8(X)                  \
  X(pa_kv_write_fp8)                          \
  X(pa_kv_read_fp8)                           \
  X(pa_decode_fp8_workspace_bytes)            \
  X(pa_decode_fp8)                            \
  X(pa_prefill_attention_fp8_workspace_bytes) \
  X(pa_prefill_attention_fp8)                 \
  X(pa_verify_drafts_workspace_bytes)         \
  X(pa_verify_drafts_f32)

// Those of sampled and forked decoding (bind_sampled).
#define PA_HOST_CALLS_SAMPLED(X)                 \
  X(pa_copy_blocks)                              \
  X(pa_sample_workspace_bytes)                   \
  X(pa_sample_tokens)                            \
  X(pa_sampling_probs)                           \
  X(pa_decode_scored_workspace_bytes)            \
  X(pa_decode_scored_f16)                        \
  X(pa_prefill_attention_scored_workspace_bytes) \
  X(pa_prefill_attention_scored_f16)

// The loaded library's entry points (bind).
struct Api {
#define PA_HOST_MEMBER(name) decltype(&::name) name;
  PA_HOST_CALLS(PA_HOST_MEMBER)
  PA_HOST_CALLS_FP8(PA_HOST_MEMBER)
  PA_HOST_CALLS_SAMPLED(PA_HOST_MEMBER)
#undef PA_HOST_MEMBER
} api;

#define PA_HOST_BIND(name) \
  api.name = reinterpret_cast<decltype(&::name)>(addresses[#name].cast<uintptr_t>());
void bind(const py::dict& addresses) {
  PA_HOST_CALLS(PA_HOST_BIND)
}

void bind_fp8(const py::dict& addresses) {
  PA_HOST_CALLS_FP8(PA_HOST_BIND)
}

void bind_sampled(const py::dict& addresses) {
  PA_HOST_CALLS_SAMPLED(PA_HOST_BIND)
}
#undef PA_HOST_BIND

// The tensors of plain torch.Tensor (or Parameter) objects, with no mode active
// that intercepts torch calls.
template <size_t N>
bool unpack(const Obj (&objects)[N], const Tensor* (&tensors)[N]) {
  if (at::impl::torch_function_mode_enabled() || c10::impl::TorchDispatchModeTLS::any_modes_set())
    return false;
  for (size_t i = 0; i < N; ++i) {
    if (!THPVariable_CheckExact(objects[i].ptr())) return false;
    tensors[i] = &THPVariable_Unpack(objects[i].ptr());
  }
  return true;
}

// Plain strided CUDA tensors of one type on one device.
bool plain(const Tensor& t, c10::ScalarType type, c10::Device dev) {
  constexpr c10::DispatchKeySet wrappers({c10::DispatchKey::Python, c10::DispatchKey::Functionalize,
                                          c10::DispatchKey::FuncTorchBatched,
                                          c10::DispatchKey::FuncTorchGradWrapper,
                                          c10::DispatchKey::Conjugate, c10::DispatchKey::Negative});
  return t.defined() && t.is_cuda() && t.device() == dev && t.scalar_type() == type &&
         t.layout() == c10::kStrided && !t.key_set().has_any(wrappers) && !t.is_nested();
}

bool current(c10::Device dev) {
  return c10::impl::getDeviceGuardImpl(c10::DeviceType::CUDA)->getDevice() == dev;
}

// Rows [rows, heads, dim] of a [rows, heads, dim] or [rows, heads, 1, dim]
// tensor: whether it is one, and its strides.
bool rows3(const Tensor& t, int64_t rows, int64_t heads, int64_t dim, int64_t (&st)[3]) {
  const int last = t.dim() - 1;
  if (last != 2 && !(last == 3 && t.size(2) == 1)) return false;
  if (t.size(0) != rows || t.size(1) != heads || t.size(last) != dim) return false;
  st[0] = t.stride(0);
  st[1] = t.stride(1);
  st[2] = t.stride(last);
  return true;
}

bool rows2(const Tensor& t, int64_t rows, int64_t dim, int64_t (&st)[2]) {
  const int last = t.dim() - 1;
  if (last != 1 && !(last == 2 && t.size(1) == 1)) return false;
  if (t.size(0) != rows || t.size(last) != dim) return false;
  st[0] = t.stride(0);
  st[1] = t.stride(last);
  return true;
}

// Unit head_dim stride, 8-element aligned strides and a 16-byte aligned base.
bool rows16(const Tensor& t, const int64_t (&st)[3]) {
  return st[2] == 1 && st[0] % 8 == 0 && st[1] % 8 == 0 && (uintptr_t)t.data_ptr() % 16 == 0;
}

// What the three calls share: pools, tables, lengths and the sizes.
struct Call {
  int64_t n, hq, hkv, d, bs, blocks, width;
  int64_t ks[4], vs[4], bts[2];

  bool fill(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& bt,
            const Tensor& lens) {
    const c10::Device dev = q.device();
    if (!plain(q, at::kHalf, dev) || !plain(k, at::kHalf, dev) || !plain(v, at::kHalf, dev) ||
        !plain(bt, at::kInt, dev) || !plain(lens, at::kInt, dev) || !current(dev))
      return false;
    if (k.dim() != 4 || k.sizes() != v.sizes() || bt.dim() != 2 || lens.dim() != 1 || q.dim() < 3)
      return false;
    n = q.size(0);
    hq = q.size(1);
    blocks = k.size(0);
    bs = k.size(1);
    hkv = k.size(2);
    d = k.size(3);
    width = bt.size(1);
    // Sizes the C ABI takes as int.
    for (int64_t x : {n, hq, hkv, d, bs, blocks, width})
      if (x <= 0 || x > 0x7fffffff) return false;
    // The C ABI reads lengths at unit stride, as the Python call passes them.
    if (hq % hkv || bt.size(0) != n || lens.size(0) != n) return false;
    for (int i = 0; i < 4; ++i) {
      ks[i] = k.stride(i);
      vs[i] = v.stride(i);
    }
    bts[0] = bt.stride(0);
    bts[1] = bt.stride(1);
    return true;
  }
};

// The caller's zero-initialised workspace of this (device, stream), if large enough.
bool workspace(const Tensor& ws, c10::Device dev, size_t need, void*& ptr) {
  ptr = nullptr;
  if (need == 0) return true;
  if (!ws.defined() || ws.device() != dev || ws.nbytes() < need) return false;
  ptr = ws.data_ptr();
  return true;
}

py::object done(int status, const Tensor& out) {
  if (status == PA_OK) return py::cast(out);
  return status == PA_ERR_HIP ? py::object(py::int_(status)) : py::object(py::none());
}

py::object decode(Obj q_, Obj k_, Obj v_, Obj bt_, Obj lens_, double scale, Obj ws_,
                  int64_t stream) {
  const Tensor* t[6];
  if (!unpack({q_, k_, v_, bt_, lens_, ws_}, t)) return py::none();
  const Tensor &q = *t[0], &k = *t[1], &v = *t[2], &bt = *t[3], &lens = *t[4], &ws = *t[5];
  Call c;
  int64_t qs[3];
  if (!c.fill(q, k, v, bt, lens) || q.dim() != 3 || !rows3(q, c.n, c.hq, c.d, qs) || !rows16(q, qs))
    return py::none();
  const size_t need = api.pa_decode_batched_workspace_bytes(c.n, c.hq, c.hkv, c.d, c.bs, c.width);
  void* wp;
  if (!workspace(ws, q.device(), need, wp)) return py::none();
  const Tensor out = at::empty_like(q);
  const int64_t os[3] = {out.stride(0), out.stride(1), out.stride(2)};
  int status;
  {
    py::gil_scoped_release release;
    status = api.pa_decode_batched_f16(q.data_ptr(), qs, k.data_ptr(), c.ks, v.data_ptr(), c.vs,
                                   (const int32_t*)bt.data_ptr(), c.bts,
                                   (const int32_t*)lens.data_ptr(), out.data_ptr(), os, c.n, c.hq,
                                   c.hkv, c.d, c.bs, c.blocks, c.width, (float)scale, wp, need,
                                   (void*)stream);
  }
  return done(status, out);
}

py::object kv_write_decode(Obj q_, Obj key_, Obj value_, Obj k_, Obj v_, Obj bt_, Obj lens_,
                           double scale, Obj ws_, int64_t stream) {
  const Tensor* t[8];
  if (!unpack({q_, key_, value_, k_, v_, bt_, lens_, ws_}, t)) return py::none();
  const Tensor &q = *t[0], &key = *t[1], &value = *t[2], &k = *t[3], &v = *t[4], &bt = *t[5],
               &lens = *t[6], &ws = *t[7];
  Call c;
  int64_t qs[3], ys[3], zs[3];
  if (!c.fill(q, k, v, bt, lens) || !plain(key, at::kHalf, q.device()) ||
      !plain(value, at::kHalf, q.device()) || !rows3(q, c.n, c.hq, c.d, qs) || !rows16(q, qs) ||
      !rows3(key, c.n, c.hkv, c.d, ys) || !rows16(key, ys) || !rows3(value, c.n, c.hkv, c.d, zs) ||
      !rows16(value, zs))
    return py::none();
  const size_t need = api.pa_decode_batched_workspace_bytes(c.n, c.hq, c.hkv, c.d, c.bs, c.width);
  void* wp;
  if (!workspace(ws, q.device(), need, wp)) return py::none();
  const Tensor out = at::empty({c.n, c.hq, c.d}, q.options());
  const int64_t os[3] = {c.hq * c.d, c.d, 1};
  int status;
  {
    py::gil_scoped_release release;
    status = api.pa_decode_kv_write_batched_f16(
        q.data_ptr(), qs, key.data_ptr(), ys, value.data_ptr(), zs, k.data_ptr(), c.ks,
        v.data_ptr(), c.vs, (const int32_t*)bt.data_ptr(), c.bts, (const int32_t*)lens.data_ptr(),
        out.data_ptr(), os, c.n, c.hq, c.hkv, c.d, c.bs, c.blocks, c.width, (float)scale, wp, need,
        (void*)stream);
  }
  return done(status, out);
}

py::object rope_decode(Obj q_, Obj key_, Obj value_, Obj cos_, Obj sin_, Obj k_, Obj v_, Obj bt_,
                       Obj lens_, double scale, Obj ws_, int64_t stream) {
  const Tensor* t[10];
  if (!unpack({q_, key_, value_, cos_, sin_, k_, v_, bt_, lens_, ws_}, t)) return py::none();
  const Tensor &q = *t[0], &key = *t[1], &value = *t[2], &cos = *t[3], &sin = *t[4], &k = *t[5],
               &v = *t[6], &bt = *t[7], &lens = *t[8], &ws = *t[9];
  Call c;
  int64_t qs[3], ys[3], zs[3], cs[2], ss[2];
  if (!c.fill(q, k, v, bt, lens) || !plain(key, at::kHalf, q.device()) ||
      !plain(value, at::kHalf, q.device()) || !plain(cos, at::kHalf, q.device()) ||
      !plain(sin, at::kHalf, q.device()) || c.d % 2 || !rows3(q, c.n, c.hq, c.d, qs) ||
      !rows3(key, c.n, c.hkv, c.d, ys) || !rows3(value, c.n, c.hkv, c.d, zs) ||
      !rows2(cos, c.n, c.d, cs) || !rows2(sin, c.n, c.d, ss))
    return py::none();
  const size_t need =
      api.pa_decode_rope_batched_workspace_bytes(c.n, c.hq, c.hkv, c.d, c.bs, c.width);
  void* wp;
  if (!workspace(ws, q.device(), need, wp)) return py::none();
  const Tensor out = at::empty({c.n, c.hq, c.d}, q.options());
  const int64_t os[3] = {c.hq * c.d, c.d, 1};
  int status;
  {
    py::gil_scoped_release release;
    status = api.pa_decode_rope_batched_f16(
        q.data_ptr(), qs, key.data_ptr(), ys, value.data_ptr(), zs, cos.data_ptr(), cs,
        sin.data_ptr(), ss, k.data_ptr(), c.ks, v.data_ptr(), c.vs, (const int32_t*)bt.data_ptr(),
        c.bts, (const int32_t*)lens.data_ptr(), out.data_ptr(), os, c.n, c.hq, c.hkv, c.d, c.bs,
        c.blocks, c.width, (float)scale, wp, need, (void*)stream);
  }
  return done(status, out);
}

// ---- the 8-bit pool ----

// Fewer than two entries, or unit stride.
bool packed(const Tensor& t) { return t.dim() == 1 && (t.size(0) < 2 || t.stride(0) == 1); }

// What the calls on the 8-bit pool share: pools, scales, tables, lengths and the sizes.
struct Pool8 {
  int64_t n, hkv, d, bs, blocks, width;
  int64_t ks[4], vs[4], kss[2], vss[2], bts[2];

  bool fill(const Tensor& k, const Tensor& v, const Tensor& kscale, const Tensor& vscale,
            const Tensor& bt, const Tensor& lens) {
    const c10::Device dev = k.device();
    if (!plain(k, at::kFloat8_e4m3fn, dev) || !plain(v, at::kFloat8_e4m3fn, dev) ||
        !plain(kscale, at::kFloat, dev) || !plain(vscale, at::kFloat, dev) ||
        !plain(bt, at::kInt, dev) || !plain(lens, at::kInt, dev) || !current(dev))
      return false;
    if (k.dim() != 4 || k.sizes() != v.sizes() || bt.dim() != 2 || !packed(lens) ||
        kscale.dim() != 2 || vscale.dim() != 2)
      return false;
    blocks = k.size(0);
    bs = k.size(1);
    hkv = k.size(2);
    d = k.size(3);
    n = lens.size(0);
    width = bt.size(1);
    for (int64_t x : {n, hkv, d, bs, blocks, width})
      if (x <= 0 || x > 0x7fffffff) return false;
    if (bt.size(0) != n || kscale.size(0) != blocks || kscale.size(1) != hkv ||
        vscale.size(0) != blocks || vscale.size(1) != hkv)
      return false;
    for (int i = 0; i < 4; ++i) {
      ks[i] = k.stride(i);
      vs[i] = v.stride(i);
    }
    for (int i = 0; i < 2; ++i) {
      kss[i] = kscale.stride(i);
      vss[i] = vscale.stride(i);
      bts[i] = bt.stride(i);
    }
    return true;
  }
};

// The first rows of sequences: n + 1 packed int32 entries.
bool starts_of(const Tensor& t, int64_t n, c10::Device dev) {
  return plain(t, at::kInt, dev) && packed(t) && t.size(0) == n + 1;
}

py::object write_fp8(Obj key_, Obj value_, Obj k_, Obj v_, Obj ks_, Obj vs_, Obj bt_, Obj lens_,
                     Obj start_, int64_t stream) {
  const Tensor* t[8];
  const Tensor* s[1] = {nullptr};
  if (!unpack({key_, value_, k_, v_, ks_, vs_, bt_, lens_}, t)) return py::none();
  if (!start_.is_none() && !unpack({start_}, s)) return py::none();
  const Tensor &key = *t[0], &value = *t[1], &k = *t[2], &v = *t[3];
  Pool8 c;
  int64_t ys[3], zs[3];
  if (!c.fill(k, v, *t[4], *t[5], *t[6], *t[7]) || !plain(key, at::kHalf, k.device()) ||
      !plain(value, at::kHalf, k.device()) || key.dim() < 3)
    return py::none();
  const int64_t rows = key.size(0);
  if (rows <= 0 || rows > 0x7fffffff || (s[0] ? key.dim() != 3 : rows != c.n)) return py::none();
  if (s[0] && !starts_of(*s[0], c.n, k.device())) return py::none();
  if (key.dim() != value.dim() || !rows3(key, rows, c.hkv, c.d, ys) ||
      !rows3(value, rows, c.hkv, c.d, zs))
    return py::none();
  int status;
  {
    py::gil_scoped_release release;
    status = api.pa_kv_write_fp8(
        key.data_ptr(), ys, value.data_ptr(), zs, k.data_ptr(), c.ks, v.data_ptr(), c.vs,
        (float*)t[4]->data_ptr(), c.kss, (float*)t[5]->data_ptr(), c.vss,
        (const int32_t*)t[6]->data_ptr(), c.bts, (const int32_t*)t[7]->data_ptr(),
        s[0] ? (const int32_t*)s[0]->data_ptr() : nullptr, c.n, rows, c.hkv, c.d, c.bs, c.blocks,
        c.width, (void*)stream);
  }
  if (status == PA_OK) return py::bool_(true);
  return status == PA_ERR_HIP ? py::object(py::int_(status)) : py::object(py::none());
}

py::object read_fp8(Obj k_, Obj v_, Obj ks_, Obj vs_, Obj bt_, Obj lens_, Obj start_, int64_t rows,
                    int64_t stream) {
  const Tensor* t[7];
  if (!unpack({k_, v_, ks_, vs_, bt_, lens_, start_}, t)) return py::none();
  const Tensor &k = *t[0], &v = *t[1];
  Pool8 c;
  if (!c.fill(k, v, *t[2], *t[3], *t[4], *t[5]) || !starts_of(*t[6], c.n, k.device()) || rows <= 0 ||
      rows > 0x7fffffff)
    return py::none();
  const Tensor key = at::empty({rows, c.hkv, c.d}, k.options().dtype(at::kHalf));
  const Tensor value = at::empty({rows, c.hkv, c.d}, k.options().dtype(at::kHalf));
  const int64_t os[3] = {c.hkv * c.d, c.d, 1};
  int status;
  {
    py::gil_scoped_release release;
    status = api.pa_kv_read_fp8(
        k.data_ptr(), c.ks, v.data_ptr(), c.vs, (const float*)t[2]->data_ptr(), c.kss,
        (const float*)t[3]->data_ptr(), c.vss, (const int32_t*)t[4]->data_ptr(), c.bts,
        (const int32_t*)t[5]->data_ptr(), (const int32_t*)t[6]->data_ptr(), key.data_ptr(), os,
        value.data_ptr(), os, c.n, rows, c.hkv, c.d, c.bs, c.blocks, c.width, (void*)stream);
  }
  if (status == PA_OK) return py::make_tuple(key, value);
  return status == PA_ERR_HIP ? py::object(py::int_(status)) : py::object(py::none());
}

py::object decode_fp8(Obj q_, Obj k_, Obj v_, Obj ks_, Obj vs_, Obj bt_, Obj lens_, double scale,
                      Obj ws_, int64_t stream) {
  const Tensor* t[8];
  if (!unpack({q_, k_, v_, ks_, vs_, bt_, lens_, ws_}, t)) return py::none();
  const Tensor &q = *t[0], &k = *t[1], &v = *t[2];
  Pool8 c;
  int64_t qs[3];
  if (!c.fill(k, v, *t[3], *t[4], *t[5], *t[6]) || !plain(q, at::kHalf, k.device()) || q.dim() != 3)
    return py::none();
  const int64_t hq = q.size(1);
  if (hq <= 0 || hq > 0x7fffffff || hq % c.hkv || !rows3(q, c.n, hq, c.d, qs) || !rows16(q, qs))
    return py::none();
  const size_t need = api.pa_decode_fp8_workspace_bytes(c.n, hq, c.hkv, c.d, c.bs, c.width);
  void* wp;
  if (!workspace(*t[7], q.device(), need, wp)) return py::none();
  const Tensor out = at::empty({c.n, hq, c.d}, q.options());
  const int64_t os[3] = {hq * c.d, c.d, 1};
  int status;
  {
    py::gil_scoped_release release;
    status = api.pa_decode_fp8(
        q.data_ptr(), qs, k.data_ptr(), c.ks, v.data_ptr(), c.vs, (const float*)t[3]->data_ptr(),
        c.kss, (const float*)t[4]->data_ptr(), c.vss, (const int32_t*)t[5]->data_ptr(), c.bts,
        (const int32_t*)t[6]->data_ptr(), out.data_ptr(), os, c.n, hq, c.hkv, c.d, c.bs, c.blocks,
        c.width, (float)scale, wp, need, (void*)stream);
  }
  return done(status, out);
}

py::object prefill_fp8(Obj q_, Obj k_, Obj v_, Obj ks_, Obj vs_, Obj bt_, Obj lens_, Obj start_,
                       int64_t most, double scale, Obj ws_, int64_t stream) {
  const Tensor* t[9];
  if (!unpack({q_, k_, v_, ks_, vs_, bt_, lens_, start_, ws_}, t)) return py::none();
  const Tensor &q = *t[0], &k = *t[1], &v = *t[2];
  Pool8 c;
  int64_t qs[3];
  if (!c.fill(k, v, *t[3], *t[4], *t[5], *t[6]) || !plain(q, at::kHalf, k.device()) || q.dim() != 3 ||
      !starts_of(*t[7], c.n, k.device()))
    return py::none();
  const int64_t rows = q.size(0), hq = q.size(1);
  for (int64_t x : {rows, hq, most})
    if (x <= 0 || x > 0x7fffffff) return py::none();
  if (hq % c.hkv || !rows3(q, rows, hq, c.d, qs) || !rows16(q, qs)) return py::none();
  const size_t need =
      api.pa_prefill_attention_fp8_workspace_bytes(c.n, hq, c.hkv, c.d, c.bs, c.width, most);
  void* wp;
  if (!workspace(*t[8], q.device(), need, wp)) return py::none();
  const Tensor out = at::empty({rows, hq, c.d}, q.options());
  const int64_t os[3] = {hq * c.d, c.d, 1};
  int status;
  {
    py::gil_scoped_release release;
    status = api.pa_prefill_attention_fp8(
        q.data_ptr(), qs, k.data_ptr(), c.ks, v.data_ptr(), c.vs, (const float*)t[3]->data_ptr(),
        c.kss, (const float*)t[4]->data_ptr(), c.vss, (const int32_t*)t[5]->data_ptr(), c.bts,
        (const int32_t*)t[6]->data_ptr(), (const int32_t*)t[7]->data_ptr(), most, out.data_ptr(),
        os, c.n, rows, hq, c.hkv, c.d, c.bs, c.blocks, c.width, (float)scale, wp, need,
        (void*)stream);
  }
  return done(status, out);
}

// ---- drafts ----

py::object verify(Obj p_, Obj q_, Obj ids_, Obj u_, Obj next_, Obj counts_, Obj ws_,
                  int64_t stream) {
  const Tensor* t[5];
  const Tensor* draft[1] = {nullptr};
  const Tensor* counts[1] = {nullptr};
  if (!unpack({p_, ids_, u_, next_, ws_}, t)) return py::none();
  if (!q_.is_none() && !unpack({q_}, draft)) return py::none();
  if (!counts_.is_none() && !unpack({counts_}, counts)) return py::none();
  const Tensor &p = *t[0], &ids = *t[1], &u = *t[2], &next = *t[3];
  const c10::Device dev = p.device();
  if (!plain(p, at::kFloat, dev) || !plain(ids, at::kLong, dev) || !plain(u, at::kFloat, dev) ||
      !plain(next, at::kFloat, dev) || !current(dev) || p.dim() != 3 || ids.dim() != 2 ||
      u.dim() != 2 || !packed(next))
    return py::none();
  const int64_t n = p.size(0), k = p.size(1) - 1, vocab = p.size(2);
  for (int64_t x : {n, k, vocab})
    if (x <= 0 || x > 0x7fffffff) return py::none();
  if (p.stride(2) != 1 || ids.size(0) != n || ids.size(1) != k || u.sizes() != ids.sizes() ||
      next.size(0) != n)
    return py::none();
  if (draft[0] && (!plain(*draft[0], at::kFloat, dev) || draft[0]->dim() != 3 ||
                   draft[0]->size(0) != n || draft[0]->size(1) != k || draft[0]->size(2) != vocab ||
                   draft[0]->stride(2) != 1))
    return py::none();
  if (counts[0] && (!plain(*counts[0], at::kInt, dev) || !packed(*counts[0]) || counts[0]->size(0) != n))
    return py::none();
  const size_t need = api.pa_verify_drafts_workspace_bytes(n, vocab);
  void* wp;
  if (!workspace(*t[4], dev, need, wp)) return py::none();
  const Tensor tokens = at::empty({n, k + 1}, ids.options());
  const Tensor accepted = at::empty({n}, ids.options().dtype(at::kInt));
  const int64_t ps[3] = {p.stride(0), p.stride(1), 1};
  int64_t qs[3] = {0, 0, 1};
  if (draft[0]) {
    qs[0] = draft[0]->stride(0);
    qs[1] = draft[0]->stride(1);
  }
  const int64_t is[2] = {ids.stride(0), ids.stride(1)}, us[2] = {u.stride(0), u.stride(1)};
  int status;
  {
    py::gil_scoped_release release;
    status = api.pa_verify_drafts_f32(
        (const float*)p.data_ptr(), ps, draft[0] ? (const float*)draft[0]->data_ptr() : nullptr, qs,
        (const int64_t*)ids.data_ptr(), is, (const float*)u.data_ptr(), us,
        (const float*)next.data_ptr(),
        counts[0] ? (const int32_t*)counts[0]->data_ptr() : nullptr, (int64_t*)tokens.data_ptr(),
        (int32_t*)accepted.data_ptr(), n, k, vocab, wp, need, (void*)stream);
  }
  if (status == PA_OK) return py::make_tuple(tokens, accepted);
  return status == PA_ERR_HIP ? py::object(py::int_(status)) : py::object(py::none());
}

// ---- scored attention ----

// Packed int32 (or fp32) entries, or None.
bool entries(Obj x, const Tensor* (&t)[1], c10::ScalarType type, int64_t n, c10::Device dev) {
  if (x.is_none()) {
    t[0] = nullptr;
    return true;
  }
  return unpack({x}, t) && plain(*t[0], type, dev) && packed(*t[0]) && t[0]->size(0) == n;
}
template <typename T>
const T* data(const Tensor* t) { return t ? (const T*)t->data_ptr() : nullptr; }

// (A window of the table's length or more is none.)
int window_of(int64_t window, const Call& c) { return window < c.width * c.bs ? (int)window : 0; }

py::object decode_scored(Obj q_, Obj k_, Obj v_, Obj bt_, Obj lens_, double scale, double softcap,
                         Obj slopes_, int64_t window, Obj starts_, Obj ws_, int64_t stream) {
  const Tensor* t[6];
  const Tensor *slopes[1], *starts[1];
  if (!unpack({q_, k_, v_, bt_, lens_, ws_}, t)) return py::none();
  const Tensor &q = *t[0], &k = *t[1], &v = *t[2], &bt = *t[3], &lens = *t[4];
  Call c;
  int64_t qs[3];
  if (!c.fill(q, k, v, bt, lens) || q.dim() != 3 || !rows3(q, c.n, c.hq, c.d, qs) ||
      !rows16(q, qs) || !packed(lens) || window < 0 ||
      !entries(slopes_, slopes, at::kFloat, c.hq, q.device()) ||
      !entries(starts_, starts, at::kInt, c.n, q.device()))
    return py::none();
  const int win = window_of(window, c);
  const size_t need =
      api.pa_decode_scored_workspace_bytes(c.n, c.hq, c.hkv, c.d, c.bs, c.width, win);
  void* wp;
  if (!workspace(*t[5], q.device(), need, wp)) return py::none();
  const Tensor out = at::empty({c.n, c.hq, c.d}, q.options());
  const int64_t os[3] = {c.hq * c.d, c.d, 1};
  int status;
  {
    py::gil_scoped_release release;
    status = api.pa_decode_scored_f16(
        q.data_ptr(), qs, k.data_ptr(), c.ks, v.data_ptr(), c.vs, (const int32_t*)bt.data_ptr(),
        c.bts, (const int32_t*)lens.data_ptr(), out.data_ptr(), os, c.n, c.hq, c.hkv, c.d, c.bs,
        c.blocks, c.width, (float)scale, (float)softcap, data<float>(slopes[0]), 1, win,
        data<int32_t>(starts[0]), wp, need, (void*)stream);
  }
  return done(status, out);
}

py::object prefill_scored(Obj q_, Obj k_, Obj v_, Obj bt_, Obj lens_, Obj start_, int64_t most,
                          double scale, double softcap, Obj slopes_, int64_t window, Obj starts_,
                          Obj ends_, Obj ws_, int64_t stream) {
  const Tensor* t[7];
  const Tensor *slopes[1], *starts[1], *ends[1];
  if (!unpack({q_, k_, v_, bt_, lens_, start_, ws_}, t)) return py::none();
  const Tensor &q = *t[0], &k = *t[1], &v = *t[2], &bt = *t[3], &lens = *t[4];
  const c10::Device dev = q.device();
  if (!plain(q, at::kHalf, dev) || !plain(k, at::kHalf, dev) || !plain(v, at::kHalf, dev) ||
      !plain(bt, at::kInt, dev) || !plain(lens, at::kInt, dev) || !current(dev) || q.dim() != 3 ||
      k.dim() != 4 || k.sizes() != v.sizes() || bt.dim() != 2 || !packed(lens))
    return py::none();
  Call c;
  c.n = lens.size(0);
  c.hq = q.size(1);
  c.blocks = k.size(0);
  c.bs = k.size(1);
  c.hkv = k.size(2);
  c.d = k.size(3);
  c.width = bt.size(1);
  const int64_t rows = q.size(0);
  for (int64_t x : {c.n, c.hq, c.hkv, c.d, c.bs, c.blocks, c.width, rows, most})
    if (x <= 0 || x > 0x7fffffff) return py::none();
  int64_t qs[3];
  if (c.hq % c.hkv || bt.size(0) != c.n || !starts_of(*t[5], c.n, dev) ||
      !rows3(q, rows, c.hq, c.d, qs) || !rows16(q, qs) || window < 0 ||
      !entries(slopes_, slopes, at::kFloat, c.hq, dev) ||
      !entries(starts_, starts, at::kInt, rows, dev) || !entries(ends_, ends, at::kInt, rows, dev))
    return py::none();
  for (int i = 0; i < 4; ++i) {
    c.ks[i] = k.stride(i);
    c.vs[i] = v.stride(i);
  }
  c.bts[0] = bt.stride(0);
  c.bts[1] = bt.stride(1);
  const int win = window_of(window, c);
  const size_t need = api.pa_prefill_attention_scored_workspace_bytes(
      c.n, c.hq, c.hkv, c.d, c.bs, c.width, most, win, ends[0] != nullptr);
  void* wp;
  if (!workspace(*t[6], dev, need, wp)) return py::none();
  const Tensor out = at::empty({rows, c.hq, c.d}, q.options());
  const int64_t os[3] = {c.hq * c.d, c.d, 1};
  int status;
  {
    py::gil_scoped_release release;
    status = api.pa_prefill_attention_scored_f16(
        q.data_ptr(), qs, k.data_ptr(), c.ks, v.data_ptr(), c.vs, (const int32_t*)bt.data_ptr(),
        c.bts, (const int32_t*)lens.data_ptr(), (const int32_t*)t[5]->data_ptr(), most,
        out.data_ptr(), os, c.n, rows, c.hq, c.hkv, c.d, c.bs, c.blocks, c.width, (float)scale,
        (float)softcap, data<float>(slopes[0]), 1, win, data<int32_t>(starts[0]),
        data<int32_t>(ends[0]), wp, need, (void*)stream);
  }
  return done(status, out);
}

// ---- pool blocks ----

py::object copy_blocks(Obj src_, Obj dst_, const py::list& caches, int64_t stream) {
  const Tensor* t[2];
  if (!unpack({src_, dst_}, t)) return py::none();
  const Tensor &src = *t[0], &dst = *t[1];
  const c10::Device dev = src.device();
  if (!plain(src, at::kInt, dev) || !plain(dst, at::kInt, dev) || !current(dev) || src.dim() != 1 ||
      dst.dim() != 1 || src.size(0) != dst.size(0))
    return py::none();
  constexpr size_t most = 1024;
  const size_t n = caches.size();
  if (n == 0 || n > most) return py::none();
  void* bases[most];
  int64_t strides[most], bytes[most], blocks = 0;
  for (size_t i = 0; i < n; ++i) {
    const Tensor* c[1];
    if (!unpack({caches[i]}, c)) return py::none();
    const Tensor& x = *c[0];
    if (!plain(x, x.scalar_type(), dev) || x.dim() < 1) return py::none();
    if (i == 0) blocks = x.size(0);
    if (x.size(0) != blocks || blocks <= 0) return py::none();
    int64_t inner = 1;  // elements of a block, which lie side by side
    for (int64_t d = x.dim() - 1; d > 0; --d) {
      if (x.size(d) != 1 && x.stride(d) != inner) return py::none();
      inner *= x.size(d);
    }
    const int64_t step = blocks > 1 ? x.stride(0) : inner;
    if (step < inner) return py::none();
    bases[i] = x.data_ptr();
    strides[i] = step * x.element_size();
    bytes[i] = inner * x.element_size();
  }
  if (src.size(0) > 0x7fffffff || blocks > 0x7fffffff) return py::none();
  int status;
  {
    py::gil_scoped_release release;
    status = api.pa_copy_blocks(bases, strides, bytes, (int)n, (const int32_t*)src.data_ptr(),
                                src.stride(0), (const int32_t*)dst.data_ptr(), dst.stride(0),
                                (int)src.size(0), (int)blocks, (void*)stream);
  }
  if (status == PA_OK) return py::bool_(true);
  return status == PA_ERR_HIP ? py::object(py::int_(status)) : py::object(py::none());
}

// ---- sampling ----

// A setting of each sequence, or a number for all.
template <typename T>
struct Setting {
  const T* each = nullptr;
  T all = 0;

  bool fill(Obj x, int64_t seqs, c10::Device dev) {
    constexpr bool whole = std::is_same_v<T, int>;
    if (PyLong_CheckExact(x.ptr())) {
      int overflow = 0;
      const long long v = PyLong_AsLongLongAndOverflow(x.ptr(), &overflow);
      if (overflow || v < -0x7fffffffLL || v > 0x7fffffffLL) return false;
      all = (T)v;
      return true;
    }
    if (PyFloat_CheckExact(x.ptr())) {
      all = (T)PyFloat_AS_DOUBLE(x.ptr());
      return !whole;
    }
    const Tensor* t[1];
    if (!unpack({x}, t)) return false;
    if (!plain(*t[0], whole ? at::kInt : at::kFloat, dev) || !packed(*t[0]) || t[0]->size(0) != seqs)
      return false;
    each = (const T*)t[0]->data_ptr();
    return true;
  }
};

// Logits [seqs, vocab] or [seqs, rows, vocab] and their settings.
struct Logits {
  int64_t seqs, rows, vocab, st[3];
  int type;
  Setting<float> temperature, top_p, min_p;
  Setting<int> top_k;

  bool fill(const Tensor& x, Obj t, Obj k, Obj p, Obj m) {
    const c10::Device dev = x.device();
    if (x.scalar_type() == at::kHalf) type = PA_F16;
    else if (x.scalar_type() == at::kBFloat16) type = PA_BF16;
    else if (x.scalar_type() == at::kFloat) type = PA_F32;
    else return false;
    if (!plain(x, x.scalar_type(), dev) || !current(dev) || (x.dim() != 2 && x.dim() != 3)) return false;
    seqs = x.size(0);
    rows = x.dim() == 3 ? x.size(1) : 1;
    vocab = x.size(-1);
    for (int64_t n : {seqs, rows, vocab})
      if (n <= 0 || n > 0x7fffffff) return false;
    st[0] = x.stride(0);
    st[1] = x.dim() == 3 ? x.stride(1) : 0;
    st[2] = x.stride(-1);
    return st[2] == 1 && temperature.fill(t, seqs, dev) && top_k.fill(k, seqs, dev) &&
           top_p.fill(p, seqs, dev) && min_p.fill(m, seqs, dev);
  }
};

py::object sample(Obj logits_, Obj u_, Obj t_, Obj k_, Obj p_, Obj m_, Obj ws_, int64_t stream) {
  const Tensor* t[3];
  if (!unpack({logits_, u_, ws_}, t)) return py::none();
  const Tensor &x = *t[0], &u = *t[1];
  Logits c;
  if (!c.fill(x, t_, k_, p_, m_) || !plain(u, at::kFloat, x.device()) || u.dim() != x.dim() - 1 ||
      u.size(0) != c.seqs || (u.dim() == 2 && u.size(1) != c.rows))
    return py::none();
  const int64_t us[2] = {u.stride(0), u.dim() == 2 ? u.stride(1) : 0};
  const size_t need = api.pa_sample_workspace_bytes(c.seqs, c.rows, c.vocab);
  void* wp;
  if (!workspace(*t[2], x.device(), need, wp)) return py::none();
  const Tensor tokens = at::empty(u.sizes(), u.options().dtype(at::kLong));
  int status;
  {
    py::gil_scoped_release release;
    status = api.pa_sample_tokens(
        x.data_ptr(), c.type, c.st, (const float*)u.data_ptr(), us, c.temperature.each,
        c.temperature.all, c.top_k.each, c.top_k.all, c.top_p.each, c.top_p.all, c.min_p.each,
        c.min_p.all, (int64_t*)tokens.data_ptr(), c.seqs, c.rows, c.vocab, wp, need, (void*)stream);
  }
  return done(status, tokens);
}

py::object probabilities(Obj logits_, Obj t_, Obj k_, Obj p_, Obj m_, Obj ws_, int64_t stream) {
  const Tensor* t[2];
  if (!unpack({logits_, ws_}, t)) return py::none();
  const Tensor& x = *t[0];
  Logits c;
  if (!c.fill(x, t_, k_, p_, m_)) return py::none();
  const size_t need = api.pa_sample_workspace_bytes(c.seqs, c.rows, c.vocab);
  void* wp;
  if (!workspace(*t[1], x.device(), need, wp)) return py::none();
  const Tensor probs = at::empty(x.sizes(), x.options().dtype(at::kFloat));
  int status;
  {
    py::gil_scoped_release release;
    status = api.pa_sampling_probs(
        x.data_ptr(), c.type, c.st, c.temperature.each, c.temperature.all, c.top_k.each, c.top_k.all,
        c.top_p.each, c.top_p.all, c.min_p.each, c.min_p.all, (float*)probs.data_ptr(), c.seqs,
        c.rows, c.vocab, wp, need, (void*)stream);
  }
  return done(status, probs);
}

}  // namespace

PYBIND11_MODULE(_pa_host, m) {
  py::list calls, calls_fp8, calls_sampled;
#define PA_HOST_NAME(name) calls.append(#name);
  PA_HOST_CALLS(PA_HOST_NAME)
#undef PA_HOST_NAME
#define PA_HOST_NAME(name) calls_fp8.append(#name);
  PA_HOST_CALLS_FP8(PA_HOST_NAME)
#undef PA_HOST_NAME
#define PA_HOST_NAME(name) calls_sampled.append(#name);
  PA_HOST_CALLS_SAMPLED(PA_HOST_NAME)
#undef PA_HOST_NAME
  m.attr("ABI_VERSION") = PA_ABI_VERSION;  // of the argument lists compiled in here
  m.attr("CALLS") = py::tuple(calls);
  m.attr("CALLS_FP8") = py::tuple(calls_fp8);
  m.attr("CALLS_SAMPLED") = py::tuple(calls_sampled);
  m.def("bind", &bind);
  m.def("bind_fp8", &bind_fp8);
  m.def("bind_sampled", &bind_sampled);
  m.def("decode", &decode);
  m.def("kv_write_decode", &kv_write_decode);
  m.def("rope_decode", &rope_decode);
  m.def("write_fp8", &write_fp8);
  m.def("read_fp8", &read_fp8);
  m.def("decode_fp8", &decode_fp8);
  m.def("prefill_fp8", &prefill_fp8);
  m.def("verify", &verify);
  m.def("decode_scored", &decode_scored);
  m.def("prefill_scored", &prefill_scored);
  m.def("copy_blocks", &copy_blocks);
  m.def("sample", &sample);
  m.def("probabilities", &probabilities);
}
