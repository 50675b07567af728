// fa_native_layer.cpp — C++ binding of the operators around the attention call (fa_rope.hip,
// fa_paged.hip), part of the _fa_native module (host code only).
//
// Their kernels take 3 to 30 us in a decoding step or a layer's training step; the Python op
// layer's checks, allocations and ctypes call take 13 to 20 us beside them, and a Python
// autograd Function another 100 us for its backward. Each function here serves a plain call:
// it makes every check of the public function that the call has to pass, well inside its
// bounds, and launches; for any other call it returns None, and Python then checks it one
// rule at a time to word its error or choose its path (rotary.py, paged.py).
#include <torch/extension.h>

#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <array>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <optional>
#include <stdexcept>
#include <string>
#include <vector>

#include "fa_native_layer.hpp"

namespace {

using Ptr = void*;
using CPtr = const void*;
using I64 = int64_t;

using Rope = int (*)(CPtr, CPtr, Ptr, Ptr, CPtr, CPtr, CPtr, CPtr, CPtr, const I64*, I64, I64, I64,
                     I64, I64, I64, I64, float, int, Ptr);
using RopeBwd = int (*)(CPtr, CPtr, CPtr, CPtr, Ptr, Ptr, Ptr, Ptr, CPtr, CPtr, CPtr, CPtr, CPtr,
                        const I64*, I64, I64, I64, I64, I64, I64, I64, float, int, Ptr, I64, Ptr);
using RopeBytes = I64 (*)(I64, I64, I64, I64, I64);
using Plan = int (*)(Ptr, I64, CPtr, CPtr, CPtr, CPtr, Ptr, Ptr, Ptr, Ptr, Ptr, I64, I64, I64, I64,
                     I64, Ptr);
using Store = int (*)(CPtr, CPtr, Ptr, Ptr, CPtr, const I64*, I64, I64, I64, I64, I64, Ptr);
using PagedBytes = I64 (*)(I64, I64, I64, I64, I64, I64, I64);
using Paged = int (*)(CPtr, CPtr, CPtr, CPtr, CPtr, Ptr, const I64*, I64, I64, I64, I64, I64, I64,
                      I64, I64, float, Ptr, I64, Ptr);
using LastError = const char* (*)();

// Entry points; index 0 = fp16, 1 = bf16.
struct Entries {
  Rope rope[2];
  RopeBwd rope_bwd[2];
  RopeBytes rope_bytes;
  Plan plan;
  Store store;
  Paged paged[2];
  PagedBytes paged_bytes;
  LastError last_error;
};
Entries g = {};
bool g_ready = false;

void check(I64 code) {
  if (code != 0)
    throw std::runtime_error("libfa_gfx950 error " + std::to_string(code) + ": " +
                             std::string(g.last_error()));
}

// ---- plain tensors ----------------------------------------------------------------------

// The tensor behind a Python object, or null for what is not a plain tensor on a gfx950 GPU.
const at::Tensor* plain(py::handle h) {
  if (!THPVariable_CheckExact(h.ptr())) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(h.ptr());
  return t.is_cuda() && t.layout() == at::kStrided ? &t : nullptr;
}

// Whether a GPU is one the kernels are built for (asked once for each).
bool served(const at::Device& device) {
  static std::array<std::atomic<int>, 64> known;  // 0 not asked, 1 yes, 2 no
  const int i = device.index();
  if (i < 0 || i >= 64) return false;
  int k = known[i].load(std::memory_order_relaxed);
  if (k == 0) {
    hipDeviceProp_t p;
    if (hipGetDeviceProperties(&p, i) != hipSuccess) return false;
    k = std::strncmp(p.gcnArchName, "gfx950", 6) == 0 ? 1 : 2;
    known[i].store(k, std::memory_order_relaxed);
  }
  return k == 1;
}

int elem_index(const at::Tensor& t) {  // -1: not a type of the kernels
  return t.scalar_type() == at::kHalf ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : -1;
}

bool is_int32(const at::Tensor& t, const at::Device& device, int dim) {
  return t.scalar_type() == at::kInt && t.device() == device && t.dim() == dim;
}

bool all_positive(const at::Tensor& t, I64 most) {
  for (const I64 n : t.sizes())
    if (n < 1 || n > most) return false;
  return true;
}

bool address16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// Whether the kernels read t's rows as they stand (_ops._readable).
bool readable(const at::Tensor& t) {
  const int last = (int)t.dim() - 1;
  if (t.is_neg() || t.stride(last) != 1 || !address16(t)) return false;
  for (int i = 0; i < last; ++i)
    if (t.size(i) > 1 && (t.stride(i) % 8 != 0 || t.stride(i) >= I64{1} << 40)) return false;
  return true;
}

at::Tensor aligned(const at::Tensor& t) {
  const at::Tensor c = t.resolve_neg().contiguous();
  return address16(c) ? c : c.clone(at::MemoryFormat::Contiguous);
}
at::Tensor operand(const at::Tensor& t) { return readable(t) ? t : aligned(t); }

I64 stride_of(const at::Tensor& t, int i) { return t.size(i) == 1 ? 0 : t.stride(i); }

Ptr stream_of(const at::Tensor& t) {
  return static_cast<Ptr>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

Ptr pointer(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

at::Tensor bytes(I64 n, const at::Tensor& like) {
  if (n < 0) check(n);
  return n > 0 ? at::empty({n}, like.options().dtype(at::kByte).requires_grad(false)) : at::Tensor();
}

void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

bool wants_grad(const at::Tensor& t) { return t.defined() && t.requires_grad(); }

// ---- norm and rotation ------------------------------------------------------------------

constexpr int kInterleaved = 1, kWeightF32 = 2, kPositionsI64 = 4;  // FA_ROPE_*

// What both directions pass on besides the rows.
struct RopeTables {
  at::Tensor cos, sin, qw, kw, positions;
  float eps;
  int flags;

  RopeTables(const at::Tensor& c, const at::Tensor& s, const at::Tensor& q_weight,
             const at::Tensor& k_weight, const at::Tensor& pos, double e, bool interleaved)
      : cos(aligned(c)), sin(aligned(s)), positions(pos), eps((float)e),
        flags(interleaved ? kInterleaved : 0) {
    if (q_weight.defined()) {
      qw = q_weight.resolve_neg().contiguous();
      kw = k_weight.resolve_neg().contiguous();
      if (qw.scalar_type() == at::kFloat) flags |= kWeightF32;
    }
    if (pos.defined() && pos.scalar_type() == at::kLong) flags |= kPositionsI64;
  }
  void position_strides(I64* s) const {
    s[0] = s[1] = 0;
    if (!positions.defined()) return;
    const int d = (int)positions.dim();
    s[1] = positions.stride(d - 1);
    if (d == 2) s[0] = positions.stride(0);
  }
};

void row_strides(const at::Tensor& t, I64* s) {
  for (int i = 0; i < 3; ++i) s[i] = stride_of(t, i);
}

std::pair<at::Tensor, at::Tensor> rope_forward(const at::Tensor& query, const at::Tensor& key,
                                               const RopeTables& r) {
  const at::Tensor q = operand(query), k = operand(key);
  at::Tensor q_out = at::empty(q.sizes(), q.options().requires_grad(false));
  at::Tensor k_out = at::empty(k.sizes(), k.options().requires_grad(false));
  I64 s[8];
  row_strides(q, s);
  row_strides(k, s + 3);
  r.position_strides(s + 6);
  check(g.rope[elem_index(q)](
      q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), r.cos.data_ptr(),
      r.sin.data_ptr(), pointer(r.positions), pointer(r.qw), pointer(r.kw), s, q.size(0), q.size(1),
      k.size(1), q.size(2), q.size(3), 2 * r.cos.size(1), r.cos.size(0), r.eps, r.flags,
      stream_of(q)));
  return {q_out, k_out};
}

// A tensor that may be left out, as torch's Function takes it.
using Maybe = std::optional<at::Tensor>;
Maybe maybe(const at::Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }

class QkNormRope : public torch::autograd::Function<QkNormRope> {
 public:
  static torch::autograd::variable_list forward(
      torch::autograd::AutogradContext* ctx, const at::Tensor& query, const at::Tensor& key,
      const Maybe& q_weight, const Maybe& k_weight, const at::Tensor& cos, const at::Tensor& sin,
      const Maybe& positions, double eps, bool interleaved) {
    const at::Tensor qw = q_weight.value_or(at::Tensor()), kw = k_weight.value_or(at::Tensor());
    const at::Tensor pos = positions.value_or(at::Tensor());
    const bool norm = qw.defined();
    ctx->save_for_backward({norm ? query : at::Tensor(), norm ? key : at::Tensor(), qw, kw, cos,
                            sin, pos});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    auto out = rope_forward(query, key, RopeTables(cos, sin, qw, kw, pos, eps, interleaved));
    return {out.first, out.second};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const RopeTables r(saved[4], saved[5], saved[2], saved[3], saved[6],
                       ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool());
    c10::DeviceGuard guard(grads[0].device());
    const bool norm = r.qw.defined();
    const at::Tensor gq = operand(grads[0]), gk = operand(grads[1]);
    I64 s[14] = {};
    row_strides(gq, s);
    row_strides(gk, s + 3);
    at::Tensor q, k, dw[2], ws;
    if (norm) {
      q = operand(saved[0]);
      k = operand(saved[1]);
      row_strides(q, s + 6);
      row_strides(k, s + 9);
      for (int i = 0; i < 2; ++i)
        if (ctx->needs_input_grad(2 + i))
          dw[i] = at::empty(r.qw.sizes(), r.qw.options().requires_grad(false));
    }
    r.position_strides(s + 12);
    const auto like = gq.options().requires_grad(false);
    at::Tensor dq = at::empty(gq.sizes(), like), dk = at::empty(gk.sizes(), like);
    const I64 B = gq.size(0), Hq = gq.size(1), Hkv = gk.size(1), N = gq.size(2), D = gq.size(3);
    I64 n = 0;
    if (dw[0].defined() || dw[1].defined()) {
      n = g.rope_bytes(B, Hq, Hkv, N, D);
      ws = bytes(n, gq);
    }
    check(g.rope_bwd[elem_index(gq)](
        gq.data_ptr(), gk.data_ptr(), pointer(q), pointer(k), dq.data_ptr(), dk.data_ptr(),
        pointer(dw[0]), pointer(dw[1]), r.cos.data_ptr(), r.sin.data_ptr(), pointer(r.positions),
        pointer(r.qw), pointer(r.kw), s, B, Hq, Hkv, N, D, 2 * r.cos.size(1), r.cos.size(0), r.eps,
        r.flags, pointer(ws), n, stream_of(gq)));
    torch::autograd::variable_list out = {dq, dk, dw[0], dw[1]};
    if (at::GradMode::is_enabled()) {
      // create_graph: the gradients have no derivative of their own; one that is asked for raises.
      auto error = std::make_shared<torch::autograd::DelayedError>(
          "qk_norm_rope's backward has no derivative of its own", 4);
      out = (*error)(std::move(out));
    }
    out.resize(9);
    return out;
  }
};

// A leaf keeps the stream that its gradient is accumulated on while any graph that uses it is
// alive. Where that is the default stream, a backward that is being captured would draw it into
// the capture, which it cannot take part in: that fails in ways that can end the process, so such
// a call is refused before it starts.
template <class Tensors>
void refuse_mixed_capture(const Tensors& leaves) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  for (const at::Tensor& t : leaves) {
    if (!wants_grad(t) || !t.is_cuda() || !t.is_leaf()) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!node) continue;
    const auto stream = node->stream();
    // (by id: autograd's streams pass for CUDA ones)
    if (stream && stream->id() == c10::hip::getDefaultHIPStream(t.device().index()).id())
      throw std::runtime_error(
          "qk_norm_rope is being captured into a graph while a result of an earlier call with the "
          "same leaf tensors is alive on the default stream: drop it first, or detach it");
  }
}

py::object native_rope(py::handle query, py::handle key, py::handle cos, py::handle sin,
                       py::handle q_weight, py::handle k_weight, py::handle eps,
                       py::handle positions, py::handle interleaved) {
  if (!g_ready) return py::none();
  const at::Tensor *q = plain(query), *k = plain(key), *c = plain(cos), *s = plain(sin);
  if (!q || !k || !c || !s || !PyBool_Check(interleaved.ptr()) || !PyFloat_CheckExact(eps.ptr()))
    return py::none();
  const at::Device device = q->device();
  const int e = elem_index(*q);
  constexpr I64 kMany = I64{1} << 24;
  if (e < 0 || k->scalar_type() != q->scalar_type() || k->device() != device ||
      c->device() != device || s->device() != device || q->dim() != 4 || k->dim() != 4 ||
      c->dim() != 2 || c->sizes() != s->sizes() || c->scalar_type() != at::kFloat ||
      s->scalar_type() != at::kFloat || !all_positive(*q, kMany) || !all_positive(*k, kMany) ||
      !all_positive(*c, kMany) || k->size(0) != q->size(0) || k->size(2) != q->size(2) ||
      k->size(3) != q->size(3) || wants_grad(*c) || wants_grad(*s) || !served(device))
    return py::none();
  const I64 B = q->size(0), N = q->size(2), D = q->size(3), P = c->size(0), half = c->size(1);
  if (D > 128 || D % 8 || half % 8 || 2 * half > D || q->size(1) >= 1 << 14 ||
      k->size(1) >= 1 << 14 || B * N >= I64{1} << 30)
    return py::none();
  at::Tensor qw, kw, pos;
  if (!q_weight.is_none() || !k_weight.is_none()) {
    const at::Tensor *a = plain(q_weight), *b = plain(k_weight);
    if (!a || !b || a->dim() != 1 || b->dim() != 1 || a->size(0) != D || b->size(0) != D ||
        a->device() != device || b->device() != device || a->scalar_type() != b->scalar_type() ||
        (a->scalar_type() != at::kFloat && a->scalar_type() != q->scalar_type()))
      return py::none();
    qw = *a;
    kw = *b;
  }
  if (!positions.is_none()) {
    const at::Tensor* p = plain(positions);
    if (!p || p->device() != device || p->dim() < 1 || p->dim() > 2 ||
        (p->scalar_type() != at::kInt && p->scalar_type() != at::kLong) ||
        p->size(p->dim() - 1) != N || (p->dim() == 2 && p->size(0) != B))
      return py::none();
    pos = *p;
  } else if (N > P) {
    return py::none();
  }
  const double ep = PyFloat_AS_DOUBLE(eps.ptr());
  if (!(ep >= 0.0 && ep <= 1e30)) return py::none();
  const bool inter = interleaved.ptr() == Py_True;
  c10::DeviceGuard guard(device);
  if (at::GradMode::is_enabled() &&
      (wants_grad(*q) || wants_grad(*k) || wants_grad(qw) || wants_grad(kw))) {
    refuse_mixed_capture(std::array<at::Tensor, 4>{*q, *k, qw, kw});
    const auto out = QkNormRope::apply(*q, *k, maybe(qw), maybe(kw), *c, *s, maybe(pos), ep, inter);
    return py::make_tuple(out[0], out[1]);
  }
  at::AutoDispatchBelowAutograd below;
  const auto out = rope_forward(*q, *k, RopeTables(*c, *s, qw, kw, pos, ep, inter));
  return py::make_tuple(out.first, out.second);
}

// ---- paged cache ------------------------------------------------------------------------

constexpr I64 kMaxTokens = (I64{1} << 30) - 64;  // that a row of the page table holds

// An int from Python, or -1.
I64 whole(py::handle h) {
  if (!PyLong_CheckExact(h.ptr())) return -1;
  int overflow = 0;
  const long long v = PyLong_AsLongLongAndOverflow(h.ptr(), &overflow);
  return overflow || v < 0 ? -1 : v;
}

// A page table [B, M] of pages of S tokens, rows of consecutive entries.
bool plain_table(const at::Tensor& t, I64 S) {
  return t.scalar_type() == at::kInt && t.dim() == 2 && t.size(1) > 0 && S > 0 && S % 16 == 0 &&
         S <= kMaxTokens && t.size(1) <= kMaxTokens / S && (t.stride(1) == 1 || t.size(1) == 1) &&
         t.size(0) < I64{1} << 24;
}

// n values of a one-dimensional tensor from `from` on, as a tensor of its own on its memory.
at::Tensor piece_of(const at::Tensor& t, I64 from, I64 n) {
  at::Tensor p = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(),
                                                          t.dtype());
  p.unsafeGetTensorImpl()->set_storage_offset(from);
  p.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return p;
}

py::object native_plan(py::handle table, py::handle lengths, py::handle new_tokens,
                       py::handle free_pages, py::handle page_size, py::handle num_tokens,
                       py::handle free_start) {
  if (!g_ready) return py::none();
  const at::Tensor *t = plain(table), *l = plain(lengths), *n = plain(new_tokens),
                   *f = plain(free_pages);
  const I64 S = whole(page_size), T = whole(num_tokens);
  if (!t || !l || !n || !f || T < 0 || T >= I64{1} << 30 || !plain_table(*t, S) ||
      !served(t->device()))
    return py::none();
  const at::Device device = t->device();
  const I64 B = t->size(0), M = t->size(1);
  if (!is_int32(*l, device, 1) || !is_int32(*n, device, 1) || !is_int32(*f, device, 1) ||
      l->size(0) != B || n->size(0) != B || f->size(0) >= I64{1} << 31 ||
      (B > 1 && t->stride(0) < M))
    return py::none();
  at::Tensor start;
  if (!free_start.is_none()) {
    const at::Tensor* p = plain(free_start);
    if (!p || p->scalar_type() != at::kInt || p->device() != device || p->numel() != 1)
      return py::none();
    start = *p;
  }
  c10::DeviceGuard guard(device);
  at::AutoDispatchBelowAutograd below;
  const auto i32 = t->options(), i64 = i32.dtype(at::kLong);
  const at::Tensor lc = l->contiguous(), nc = n->contiguous(), fc = f->contiguous();
  // One allocation for the four int32 results (a step's plan waits for the host otherwise).
  const at::Tensor small = at::empty({T + 2 * B + 2}, i32);
  at::Tensor slots = at::empty({T}, i64), positions = piece_of(small, 0, T);
  at::Tensor starts = piece_of(small, T, B + 1), held = piece_of(small, T + B + 1, B);
  at::Tensor free_out = piece_of(small, T + 2 * B + 1, 1);
  check(g.plan(t->data_ptr(), t->stride(0), lc.data_ptr(), nc.data_ptr(), fc.data_ptr(),
               pointer(start), slots.data_ptr(), positions.data_ptr(), starts.data_ptr(),
               held.data_ptr(), free_out.data_ptr(), B, M, S, fc.size(0), T, stream_of(*t)));
  written(*t);
  return py::make_tuple(slots, positions, starts, held, free_out);
}

// Caches that the kernels address as they stand (paged._cache_reason); false for any doubt.
bool plain_caches(const at::Tensor& k, const at::Tensor& v) {
  if (elem_index(k) < 0 || v.scalar_type() != k.scalar_type() || k.device() != v.device() ||
      k.dim() != 4 || v.sizes() != k.sizes() || v.strides() != k.strides() ||
      !all_positive(k, I64{1} << 30) || k.is_neg() || v.is_neg())
    return false;
  const I64 D = k.size(3);
  if (D > 128 || D % 8 || k.size(2) % 16 || k.stride(3) != 1 || !address16(k) || !address16(v))
    return false;
  for (int i = 0; i < 3; ++i)
    if (k.stride(i) % 8 || k.stride(i) <= 0 || k.stride(i) >= I64{1} << 40) return false;
  return k.stride(2) >= D && k.stride(2) < 1 << 25;
}

void cache_strides(const at::Tensor& t, I64* s) {
  s[0] = stride_of(t, 0);
  s[1] = stride_of(t, 1);
  s[2] = t.stride(2);
}

// True where the store was made.
bool native_store(py::handle key, py::handle value, py::handle key_cache, py::handle value_cache,
                  py::handle slots) {
  if (!g_ready) return false;
  const at::Tensor *k = plain(key), *v = plain(value), *kc = plain(key_cache),
                   *vc = plain(value_cache), *s = plain(slots);
  if (!k || !v || !kc || !vc || !s || !plain_caches(*kc, *vc) || !served(kc->device())) return false;
  const at::Device device = kc->device();
  if (kc->data_ptr() == vc->data_ptr() || k->scalar_type() != kc->scalar_type() || v->scalar_type() != kc->scalar_type() ||
      k->device() != device || v->device() != device || s->device() != device || k->dim() != 3 ||
      v->sizes() != k->sizes() || k->size(1) != kc->size(1) || k->size(2) != kc->size(3) ||
      s->scalar_type() != at::kLong || s->dim() != 1 || s->size(0) != k->size(0) ||
      k->size(0) < 1 || k->size(0) >= I64{1} << 31 || k->size(1) >= 1 << 20)
    return false;
  if (at::GradMode::is_enabled() &&
      (wants_grad(*k) || wants_grad(*v) || wants_grad(*kc) || wants_grad(*vc)))
    return false;
  c10::DeviceGuard guard(device);
  at::AutoDispatchBelowAutograd below;
  const at::Tensor kr = operand(*k), vr = operand(*v), sc = s->contiguous();
  I64 st[7] = {stride_of(kr, 0), stride_of(kr, 1), stride_of(vr, 0), stride_of(vr, 1)};
  cache_strides(*kc, st + 4);
  check(g.store(kr.data_ptr(), vr.data_ptr(), kc->data_ptr(), vc->data_ptr(), sc.data_ptr(), st,
                k->size(0), k->size(1), k->size(2), kc->size(0), kc->size(2), stream_of(*kc)));
  written(*kc);
  written(*vc);
  return true;
}

py::object native_paged(py::handle query, py::handle key_cache, py::handle value_cache,
                        py::handle table, py::handle lengths, py::handle scale,
                        py::handle enable_gqa) {
  if (!g_ready) return py::none();
  const at::Tensor *q = plain(query), *kc = plain(key_cache), *vc = plain(value_cache),
                   *t = plain(table), *l = plain(lengths);
  if (!q || !kc || !vc || !t || !l || !PyBool_Check(enable_gqa.ptr()) || !plain_caches(*kc, *vc) ||
      !plain_table(*t, kc->size(2)) || !served(q->device()))
    return py::none();
  const at::Device device = q->device();
  constexpr I64 kMany = I64{1} << 16;
  if (q->scalar_type() != kc->scalar_type() || kc->device() != device || t->device() != device ||
      q->dim() != 4 || !all_positive(*q, kMany) || q->size(3) != kc->size(3) ||
      t->size(0) != q->size(0) || !is_int32(*l, device, 1) || l->size(0) != q->size(0))
    return py::none();
  const I64 B = q->size(0), Hq = q->size(1), N = q->size(2), D = q->size(3);
  const I64 pages = kc->size(0), H = kc->size(1), S = kc->size(2), M = t->size(1);
  if (Hq % H || (Hq != H && enable_gqa.ptr() != Py_True)) return py::none();
  if (at::GradMode::is_enabled() && (wants_grad(*q) || wants_grad(*kc) || wants_grad(*vc)))
    return py::none();
  double sc = 0.0;
  if (scale.is_none()) sc = std::pow(static_cast<double>(D), -0.5);
  else if (PyFloat_CheckExact(scale.ptr())) sc = PyFloat_AS_DOUBLE(scale.ptr());
  if (!(sc >= 1e-30 && sc <= 1e30)) return py::none();
  const I64 n = g.paged_bytes(B, Hq, H, N, D, M, S);
  if (n < 0) return py::none();
  c10::DeviceGuard guard(device);
  at::AutoDispatchBelowAutograd below;
  const at::Tensor qr = operand(*q), lc = l->contiguous();
  const at::Tensor ws = bytes(n, qr);
  at::Tensor o = at::empty({B, Hq, N, D}, qr.options().requires_grad(false));
  I64 st[7];
  row_strides(qr, st);
  cache_strides(*kc, st + 3);
  st[6] = t->stride(0);
  check(g.paged[elem_index(*q)](qr.data_ptr(), kc->data_ptr(), vc->data_ptr(), t->data_ptr(),
                                lc.data_ptr(), o.data_ptr(), st, B, Hq, H, N, D, pages, M, S,
                                (float)sc, pointer(ws), n, stream_of(*q)));
  return py::cast(o);
}

// Takes the entry points' addresses, in the order of Entries.
void init_layer(const std::vector<I64>& addresses) {
  if (addresses.size() != 11)
    throw std::invalid_argument("gfx950 layer operators: 11 entry points are needed");
  for (const I64 a : addresses)
    if (a == 0) throw std::invalid_argument("gfx950 layer operators: a null entry point was passed");
  auto at = [&](int i) { return reinterpret_cast<Ptr>(static_cast<uintptr_t>(addresses[i])); };
  for (int i = 0; i < 2; ++i) {
    g.rope[i] = reinterpret_cast<Rope>(at(i));
    g.rope_bwd[i] = reinterpret_cast<RopeBwd>(at(2 + i));
    g.paged[i] = reinterpret_cast<Paged>(at(7 + i));
  }
  g.rope_bytes = reinterpret_cast<RopeBytes>(at(4));
  g.plan = reinterpret_cast<Plan>(at(5));
  g.store = reinterpret_cast<Store>(at(6));
  g.paged_bytes = reinterpret_cast<PagedBytes>(at(9));
  g.last_error = reinterpret_cast<LastError>(at(10));
  g_ready = true;
}

}  // namespace

void bind_layer(py::module_& m) {
  m.def("init_layer", &init_layer);
  m.def("qk_norm_rope", &native_rope);
  m.def("refuse_mixed_capture", &refuse_mixed_capture<std::vector<at::Tensor>>);
  m.def("paged_plan", &native_plan);
  m.def("paged_store", &native_store);
  m.def("paged_attention", &native_paged);
}
