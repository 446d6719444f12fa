// Host side of the encoder operators (ops/attention.py, ops/residual.py): plans the launches, allocates outputs and scratch from
// PyTorch's allocator on the current stream, and records the backward passes as C++ autograd nodes - in Python they cost
// two to three times the kernels of a learner step, most of it in the autograd thread.  Arguments are checked in Python
// before they get here; the kernel library's entry points are handed over as addresses (bind), so nothing here links HIP.
#include <Python.h>
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <initializer_list>
#include <map>
#include <optional>
#include <string>

#include "../hip/encoder_ops.h"

namespace py = pybind11;
using at::Tensor;
using atrihip::EncAttnArgs;
using atrihip::ResNormArgs;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

using AttnFn = int (*)(const EncAttnArgs*, ihipStream_t*);
using NormFn = int (*)(const ResNormArgs*, ihipStream_t*);
struct {
  AttnFn attn_fwd = nullptr, attn_bwd = nullptr;
  NormFn norm_fwd = nullptr, norm_bwd = nullptr;
} lib;

void bind(const std::map<std::string, uintptr_t>& entries) {
  lib.attn_fwd = reinterpret_cast<AttnFn>(entries.at("atri_enc_attn_fwd"));
  lib.attn_bwd = reinterpret_cast<AttnFn>(entries.at("atri_enc_attn_bwd"));
  lib.norm_fwd = reinterpret_cast<NormFn>(entries.at("atri_resnorm_fwd"));
  lib.norm_bwd = reinterpret_cast<NormFn>(entries.at("atri_resnorm_bwd"));
}

template <typename Fn, typename Args>
void launch(Fn fn, const Args& args, const char* name, const Tensor& on) {
  TORCH_CHECK(fn != nullptr && on.is_cuda(), name, " needs the kernel library and tensors on the GPU");
  const int rc = fn(&args, reinterpret_cast<ihipStream_t*>(c10::hip::getCurrentHIPStream(on.device().index()).stream()));
  TORCH_CHECK(rc == 0, name, " failed with code ", rc);
}

int64_t up(int64_t n, int64_t d) { return (n + d - 1) / d; }
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
float* f32(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

Tensor param(const Tensor& t) {  // fp32, contiguous, on 16 bytes
  if (!t.defined()) return t;
  Tensor p = t.detach().to(at::kFloat).contiguous();
  return aligned(p) ? p : p.clone();
}

// The kernels compute values.  A tangent would be lost without a word where no autograd node is made, and a trace would record the
// output's allocation and nothing else.
void values_only(const char* name, std::initializer_list<const Tensor*> given) {
  TORCH_CHECK(!torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(), name,
              ": cannot be traced (torch.jit.trace, make_fx): its kernels are launched outside of PyTorch's operators");
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : given)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), name, ": differentiable in reverse mode only, got a tensor with a forward-mode tangent");
}

// A leaf's gradient accumulator runs on the stream it was made on, and lives as long as a graph of that leaf does.  A captured backward
// pass would reach out to it, and the default stream cannot be part of a capture: refused while nothing is recorded yet.
void refuse_capture_beside_eager_graph(const char* name, std::initializer_list<const Tensor*> given) {
  const c10::DeviceGuard guard((*given.begin())->device());
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  for (const Tensor* t : given) {
    if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto stream = accumulator ? accumulator->stream() : std::nullopt;
    TORCH_CHECK(!stream || stream->id() != c10::hip::getDefaultHIPStream(t->device().index()).id(), name,
                ": an eager graph of one of these leaves lives, made on the default stream; a backward pass captured now would run on that stream too: drop the eager "
                "graph's tensors before the capture, or capture a call on detached leaves");
  }
}

// The gradients of a first-order node: usable as they are, an error when somebody differentiates them again.
variable_list once(variable_list grads, const char* what) {
  if (!at::GradMode::is_enabled()) return grads;
  auto error = std::make_shared<torch::autograd::DelayedError>(std::string("trying to differentiate ") + what + " twice: it is differentiable once",
                                                               static_cast<int64_t>(grads.size()));
  variable_list in;
  for (auto& g : grads) in.push_back(g.defined() ? g.detach().requires_grad_(true) : g);
  return (*error)(std::move(in));
}

// ------------------------------------------------------------------------------------------------------- attention
struct Call {
  Tensor lut, order, start, mask, qoff;
  int64_t radius = 0, cols = 0, buckets = 0, q0 = 0, maps = 1;
  double scale = 1.0;
};

// t as the kernels can read it: in place when its rows are contiguous and 16-byte aligned, else a copy.
Tensor rows(const Tensor& given) {
  Tensor t = given.detach();
  const int64_t vec = t.scalar_type() == at::kFloat ? 3 : 7;
  bool ok = t.stride(3) == 1 && aligned(t);
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) == 1 || (t.stride(i) & vec) == 0);
  if (ok) return t;
  t = t.contiguous();
  return aligned(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}

// New [B, L, heads, width] in the type and the token / batch order of t; no view, so that an output takes in-place operations.
Tensor empty_rows(const Tensor& t, int64_t heads, int64_t width) {
  const int64_t b = t.size(0), n = t.size(1);
  if (t.stride(0) < t.stride(1) && b > 1 && n > 1) return at::empty_strided({b, n, heads, width}, {heads * width, b * heads * width, width, 1}, t.options());
  return at::empty({b, n, heads, width}, t.options());
}

void strides(long long (&s)[3], const Tensor& t) {
  for (int i = 0; i < 3; ++i) s[i] = t.stride(i);
}

// Key (query) ranges per workgroup row and samples per workgroup of a launch with `groups` workgroups per sample that walk
// `steps` tiles each, on a card that holds `resident` of them at a time.
//   more than fit: every workgroup takes several samples (its bias is laid out once, loads run ahead across samples), so that
//   one round of them covers the batch;
//   fewer: the tiles are split where that shortens the rounds.  A workgroup costs its tiles and two more for its ends, a
//   split the write and join of its `partial` floats: half a tile, a tenth where they are under 1 MB and stay in L2 (one
//   token of four sequences of 8190: 21.4 us with a half, 18.7 with a tenth; 12004 rows of two maps: 324 and 331 us).
void plan(int64_t samples, int64_t groups, int64_t steps, int64_t resident, int64_t partial, int& splits, int& chunk) {
  const int64_t n = samples * groups;
  splits = 1;
  chunk = static_cast<int>(up(n, resident));
  if (chunk > 1) return;
  const double join = partial < (1 << 18) ? 0.1 : 0.5;
  const auto cost = [&](int64_t s) { return static_cast<double>(up(n * s, resident) * (up(steps, s) + 2)) + (s > 1 ? 2.0 + join * static_cast<double>(s) : 0.0); };
  double best = cost(1);
  for (int64_t s = 2; s <= std::min<int64_t>(steps, 128); ++s)
    if (cost(s) < 0.95 * best) best = cost(s), splits = static_cast<int>(s);
}

// Workgroups of one pass that the card's 256 compute units hold at a time (four waves each, one per SIMD); sums: with room for sums by position,
// also where they are not wanted, so that gradients do not depend on that.
int64_t resident(const EncAttnArgs& a, int pass, bool sums = false) {
  return 256 * atrihip::enc_workgroups(a.bf16 != 0, a.D, a.M, a.table ? a.R : -1, a.W, a.Lq, a.Lk, a.H == a.KV, pass, sums);
}

struct Sizes {
  int64_t b, lq, lk, h, kv, d, dv, maps, rows;
  bool bf16;
  int64_t n_words, n_stat, n_o32;  // floats of the three parts of what the forward pass keeps, each padded to 16 bytes
};

Sizes sizes(const Call& c, const Tensor& q, const Tensor& v, bool train, bool masked) {
  Sizes s{};
  s.b = q.size(0); s.lq = q.size(1); s.lk = v.size(1);
  s.maps = c.maps; s.h = q.size(2) / c.maps; s.kv = v.size(2); s.d = q.size(3); s.dv = v.size(3);
  s.rows = s.b * s.h * s.lq;
  s.bf16 = q.scalar_type() == at::kBFloat16;
  s.n_words = masked ? up(2 * s.b * up(s.lk, atrihip::kTile), 4) * 4 : 0;
  s.n_stat = train ? up(2 * s.maps * s.rows, 4) * 4 : 0;
  s.n_o32 = train && (s.bf16 || s.maps == 2) ? s.maps * s.rows * s.dv : 0;
  return s;
}

EncAttnArgs base_args(const Call& c, const Sizes& s, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lam) {
  EncAttnArgs a{};
  a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr();
  strides(a.qs, q); strides(a.ks, k); strides(a.vs, v);
  a.lam = f32(lam);
  if (table.defined()) {
    a.table = f32(table);
    a.lut = c.lut.data_ptr<int>();
    a.order = c.order.data_ptr<int>();
    a.start = c.start.data_ptr<int>();
    a.R = static_cast<int>(c.radius); a.W = static_cast<int>(c.cols); a.buckets = static_cast<int>(c.buckets);
  }
  if (c.qoff.defined()) a.qoff = c.qoff.data_ptr<int>();
  a.B = static_cast<int>(s.b); a.Lq = static_cast<int>(s.lq); a.Lk = static_cast<int>(s.lk);
  a.H = static_cast<int>(s.h); a.KV = static_cast<int>(s.kv); a.D = static_cast<int>(s.d); a.DV = static_cast<int>(s.dv); a.M = static_cast<int>(s.maps);
  a.q0 = static_cast<int>(c.q0);
  a.bf16 = s.bf16;
  a.splits = a.chunk = a.q_splits = a.q_chunk = a.k_splits = a.k_chunk = a.shares = 1;
  a.hist_rows = 4;
  a.scale = static_cast<float>(c.scale);
  const long long o32[4] = {s.h * s.lq * s.dv, s.dv, s.lq * s.dv, s.rows * s.dv};
  std::copy(o32, o32 + 4, a.o32s);
  return a;
}

// The output and, for a backward pass, one buffer of what it keeps: validity words (if masked), (maximum, 1 / sum) of every row
// and - unless the fp32 output itself will do - every map's output in 32 bits.
Tensor attention_forward(const Call& c, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lam, bool train, Tensor& keep) {
  const Sizes s = sizes(c, q, v, train, c.mask.defined());
  EncAttnArgs a = base_args(c, s, q, k, v, table, lam);
  Tensor out = empty_rows(q, s.h, s.dv);
  a.out = out.data_ptr();
  strides(a.os, out);
  const auto f = q.options().dtype(at::kFloat);
  if (s.n_words + s.n_stat + s.n_o32) {
    keep = at::empty({s.n_words + s.n_stat + s.n_o32}, f);
    float* at_keep = f32(keep);
    if (s.n_words) {
      a.mask = static_cast<const unsigned char*>(c.mask.data_ptr());
      a.ms[0] = c.mask.stride(0); a.ms[1] = c.mask.stride(1);
      a.words = reinterpret_cast<unsigned long long*>(at_keep);
    }
    if (s.n_stat) a.stat = at_keep + s.n_words;
    if (s.n_o32) a.o32 = at_keep + s.n_words + s.n_stat;
  }
  const bool board = atrihip::enc_board_tiles(a.W, a.Lk, a.D, a.M) > 0;  // unrolled over its tiles: never split
  const int64_t per = 64 * atrihip::enc_columns(a.W, a.Lq, a.Lk, a.D, a.M, a.bf16 != 0, atrihip::kEncForward);
  plan(s.b, s.h * up(s.lq, per), board ? 1 : up(s.lk, atrihip::kTile), resident(a, atrihip::kEncForward), s.maps * s.rows * s.dv, a.splits, a.chunk);
  Tensor part;
  if (a.splits > 1) {
    const int64_t n = a.splits * s.maps * s.rows;
    part = at::empty({n * (s.dv + 2)}, f);
    a.part_o = f32(part);
    a.part_ml = a.part_o + n * s.dv;
  }
  launch(lib.attn_fwd, a, "atri_enc_attn_fwd", q);
  return out;
}

struct Attention : torch::autograd::Function<Attention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q_, const Tensor& k_, const Tensor& v_, const std::optional<Tensor>& table_opt,
                        const std::optional<Tensor>& lam_opt, const Call& c) {
    const c10::DeviceGuard guard(q_.device());
    const Tensor table_ = table_opt.value_or(Tensor()), lam_ = lam_opt.value_or(Tensor());
    const Tensor q = rows(q_), k = rows(k_), v = rows(v_), table = param(table_), lam = param(lam_);
    Tensor keep;
    Tensor out = attention_forward(c, q, k, v, table, lam, true, keep);
    const bool own_out = c.maps == 1 && q.scalar_type() == at::kFloat;
    ctx->save_for_backward({q, k, v, table, lam, keep, own_out ? out : Tensor(), c.lut, c.order, c.start, c.qoff});
    ctx->saved_data["call"] = std::vector<int64_t>{c.radius, c.cols, c.buckets, c.q0, c.maps, c.mask.defined(),
                                                   static_cast<int64_t>(table_.defined() ? table_.scalar_type() : at::kFloat),
                                                   static_cast<int64_t>(lam_.defined() ? lam_.scalar_type() : at::kFloat)};
    ctx->saved_data["scale"] = c.scale;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) { return once(gradients(ctx, grads), "encoder attention"); }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &table = saved[3], &lam = saved[4], &keep = saved[5], &out = saved[6];
    const auto ints = ctx->saved_data["call"].toIntVector();
    Call c;
    c.lut = saved[7]; c.order = saved[8]; c.start = saved[9]; c.qoff = saved[10];
    c.radius = ints[0]; c.cols = ints[1]; c.buckets = ints[2]; c.q0 = ints[3]; c.maps = ints[4];
    c.scale = ctx->saved_data["scale"].toDouble();
    const c10::DeviceGuard guard(q.device());
    const at::NoGradGuard no_grad;
    const Tensor dout = rows(grads[0].to(q.scalar_type()));
    const Sizes s = sizes(c, q, v, true, ints[5] != 0);
    EncAttnArgs a = base_args(c, s, q, k, v, table, lam);
    // edges: q, k, v, then the table and lam where they are given
    const bool want_kv = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    const bool want_table = table.defined() && ctx->needs_input_grad(3), want_lam = lam.defined() && ctx->needs_input_grad(table.defined() ? 4 : 3);
    Tensor dq = empty_rows(q, q.size(2), s.d), dk, dv;
    a.dout = dout.data_ptr(); a.dq = dq.data_ptr();
    strides(a.gs, dout); strides(a.dqs, dq);
    if (want_kv) {  // without them the key-owned pass is left out
      dk = empty_rows(k, k.size(2), s.d);
      dv = empty_rows(v, s.kv, s.dv);
      a.dk = dk.data_ptr(); a.dv = dv.data_ptr();
      strides(a.dks, dk); strides(a.dvs, dv);
    }
    float* at_keep = f32(keep);
    if (s.n_words) a.words = reinterpret_cast<unsigned long long*>(at_keep);
    a.stat = at_keep + s.n_words;
    if (out.defined()) {
      a.o32 = f32(out);
      for (int i = 0; i < 3; ++i) a.o32s[i] = out.stride(i);
      a.o32s[3] = 0;
    } else {
      a.o32 = a.stat + s.n_stat;
    }
    const int64_t nqt = up(s.lq, 64 * atrihip::enc_columns(a.W, a.Lq, a.Lk, a.D, a.M, a.bf16 != 0, atrihip::kEncQueries));
    // shared heads take the general form of the key-owned pass
    const int64_t nkt = up(s.lk, 64 * atrihip::enc_columns(s.h == s.kv ? a.W : 0, a.Lq, a.Lk, a.D, a.M, a.bf16 != 0, atrihip::kEncKeys));
    const bool board = atrihip::enc_board_tiles(a.W, a.Lk, a.D, a.M) > 0;  // unrolled over its tiles: never split
    plan(s.b, s.h * nqt, board ? 1 : up(s.lk, atrihip::kTile), resident(a, atrihip::kEncQueries, table.defined()), s.rows * s.maps * s.d, a.q_splits, a.q_chunk);
    plan(s.b, s.kv * nkt, board && s.h == s.kv ? 1 : s.h / s.kv * up(s.lq, atrihip::kTile), resident(a, atrihip::kEncKeys),
         s.b * s.kv * s.lk * (s.maps * s.d + s.dv), a.k_splits, a.k_chunk);
    const int64_t hm = s.h * s.maps, slots = 2 * c.radius + 1, per_head = up(s.b, a.q_chunk) * a.q_splits * nqt;
    a.q_groups = per_head * s.h;
    a.shares = static_cast<int>(std::clamp<int64_t>(per_head / 16, 1, 64));
    const int64_t n_delta = up(s.maps * s.rows, 4) * 4, n_dq = a.q_splits > 1 ? a.q_splits * s.rows * s.maps * s.d : 0;
    const int64_t n_kv = want_kv && a.k_splits > 1 ? a.k_splits * s.b * s.kv * s.lk * (s.maps * s.d + s.dv) : 0;
    const int64_t n_hist = want_table ? per_head * hm * slots : 0, n_mid = want_table ? a.shares * hm * slots : 0;
    const auto f = q.options().dtype(at::kFloat);
    const int64_t n_dlam = want_lam ? per_head * s.h * 4 : 0;
    const Tensor work = at::empty({n_delta + n_dq + n_kv + n_hist + n_mid + n_dlam}, f);
    a.delta = f32(work);
    if (n_dq) a.dq_part = a.delta + n_delta;
    if (n_kv) a.kv_part = a.delta + n_delta + n_dq;
    Tensor dtable, dlam;
    if (want_table) {
      dtable = at::empty({c.buckets, hm}, f);
      a.hist = a.delta + n_delta + n_dq + n_kv;
      a.mid = a.hist + n_hist;
      a.dtable = f32(dtable);
    }
    if (want_lam) {
      dlam = at::empty({s.h}, f);
      a.dlam = f32(dlam);
      a.dlam_part = a.delta + n_delta + n_dq + n_kv + n_hist + n_mid;
    }
    launch(lib.attn_bwd, a, "atri_enc_attn_bwd", q);
    if (want_table) dtable = dtable.to(static_cast<at::ScalarType>(ints[6]));
    if (want_lam) dlam = dlam.to(static_cast<at::ScalarType>(ints[7]));
    return {dq, dk, dv, dtable, dlam, Tensor()};
  }
};

Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const std::optional<Tensor>& table, const std::optional<Tensor>& lam,
                 const std::optional<Tensor>& lut, const std::optional<Tensor>& order, const std::optional<Tensor>& start, int64_t radius, int64_t cols,
                 int64_t buckets, const std::optional<Tensor>& mask, const std::optional<Tensor>& qoff, int64_t q0, double scale) {
  const Tensor none;
  Call c;
  c.lut = lut.value_or(none); c.order = order.value_or(none); c.start = start.value_or(none);
  c.mask = mask.value_or(none); c.qoff = qoff.value_or(none);
  c.radius = radius; c.cols = cols; c.buckets = buckets; c.q0 = q0; c.scale = scale;
  c.maps = lam.has_value() ? 2 : 1;
  const Tensor t = table.value_or(none), l = lam.value_or(none);
  values_only("encoder attention", {&q, &k, &v, &t, &l});
  const bool grads = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad() || (t.defined() && t.requires_grad()) ||
                                                    (l.defined() && l.requires_grad()));
  if (grads) refuse_capture_beside_eager_graph("encoder attention", {&q, &k, &v, &t, &l});
  if (grads) return Attention::apply(q, k, v, table, lam, c);
  const c10::DeviceGuard guard(q.device());
  Tensor keep;
  return attention_forward(c, rows(q), rows(k), rows(v), param(t), param(l), false, keep);
}

// -------------------------------------------------------------------------------------------------- residual joint
Tensor flat(const Tensor& given) {  // contiguous, on 16 bytes
  if (!given.defined()) return given;
  Tensor t = given.detach().contiguous();
  return aligned(t) ? t : t.clone();
}

ResNormArgs norm_args(const Tensor& x, const Tensor& z, const Tensor& gate, const Tensor* params, double eps) {
  ResNormArgs a{};
  a.x = x.data_ptr(); a.z = z.data_ptr();
  a.gate = gate.defined() ? gate.data_ptr() : nullptr;
  a.scale = f32(params[0]); a.post_w = f32(params[1]); a.post_b = f32(params[2]); a.pre_w = f32(params[3]); a.pre_b = f32(params[4]);
  a.D = static_cast<int>(x.size(-1));
  a.N = x.numel() / a.D;
  a.gate_mode = !gate.defined() ? 0 : gate.sizes() == z.sizes() ? 2 : 1;
  a.x_bf16 = x.scalar_type() == at::kBFloat16;
  a.z_bf16 = z.scalar_type() == at::kBFloat16;
  a.eps = static_cast<float>(eps);
  return a;
}

// Workgroups of a launch: one step each while there are few rows, then `most` that walk the rest.
int norm_groups(const ResNormArgs& a, int64_t most) {
  const int lanes = atrihip::lanes_of(a.D);
  return static_cast<int>(std::clamp<int64_t>(up(a.N, atrihip::threads_of(lanes) / lanes), 1, most));
}

variable_list norm_forward(const Tensor& x, const Tensor& z, const Tensor& gate, const Tensor* params, double eps, Tensor* stats) {
  ResNormArgs a = norm_args(x, z, gate, params, eps);
  Tensor y = at::empty_like(x), h = at::empty_like(z);
  a.y = y.data_ptr(); a.h = h.data_ptr();
  if (stats) {
    *stats = at::empty({static_cast<int64_t>(a.N), 4}, x.options().dtype(at::kFloat));
    a.stats = f32(*stats);
  }
  a.groups = norm_groups(a, 2048);
  launch(lib.norm_fwd, a, "atri_resnorm_fwd", x);
  return {y, h};
}

struct GatedNormResidual : torch::autograd::Function<GatedNormResidual> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x_, const Tensor& z_, const Tensor& scale, const Tensor& post_w, const Tensor& post_b,
                               const Tensor& pre_w, const Tensor& pre_b, const std::optional<Tensor>& gate_, double eps) {
    const c10::DeviceGuard guard(x_.device());
    const Tensor x = flat(x_), z = flat(z_), gate = flat(gate_.value_or(Tensor()));
    const Tensor params[5] = {param(scale), param(post_w), param(post_b), param(pre_w), param(pre_b)};
    Tensor stats;
    variable_list out = norm_forward(x, z, gate, params, eps, &stats);
    ctx->save_for_backward({x, z, gate, stats, params[0], params[1], params[2], params[3], params[4]});
    ctx->set_materialize_grads(false);
    std::vector<int64_t> types;
    for (const Tensor& p : {scale, post_w, post_b, pre_w, pre_b}) types.push_back(static_cast<int64_t>(p.scalar_type()));
    ctx->saved_data["types"] = types;
    ctx->saved_data["eps"] = eps;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) { return once(gradients(ctx, grads), "gated_norm_residual"); }

  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &z = saved[1], &gate = saved[2], &stats = saved[3];
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(9);
    const c10::DeviceGuard guard(x.device());
    const at::NoGradGuard no_grad;
    const Tensor dy = grads[0].defined() ? flat(grads[0].to(x.scalar_type())) : Tensor();
    const Tensor dh = grads[1].defined() ? flat(grads[1].to(z.scalar_type())) : Tensor();
    ResNormArgs a = norm_args(x, z, gate, &saved[4], ctx->saved_data["eps"].toDouble());
    Tensor dx = at::empty_like(x), dz = at::empty_like(z), dgate = gate.defined() ? at::empty_like(gate) : Tensor();
    a.stats = f32(stats);
    a.dy = dy.defined() ? dy.data_ptr() : nullptr;
    a.dh = dh.defined() ? dh.data_ptr() : nullptr;
    a.dx = dx.data_ptr(); a.dz = dz.data_ptr();
    a.dgate = gate.defined() ? dgate.data_ptr() : nullptr;
    a.groups = norm_groups(a, a.D <= 512 ? 1024 : 512);  // many rows per workgroup keep the partial sums (5 rows each) small beside the rows
    const auto f = x.options().dtype(at::kFloat);
    const Tensor part = at::empty({a.groups, 5, a.D}, f), dparams = at::empty({5, a.D}, f);
    a.part = f32(part);
    a.dparams = f32(dparams);
    launch(lib.norm_bwd, a, "atri_resnorm_bwd", x);
    const auto types = ctx->saved_data["types"].toIntVector();
    variable_list all = {dx, dz};
    const auto each = dparams.unbind(0);
    for (int i = 0; i < 5; ++i) all.push_back(each[i].to(static_cast<at::ScalarType>(types[i])));
    all.push_back(dgate);
    all.emplace_back();
    return all;
  }
};

std::pair<Tensor, Tensor> gated_norm_residual(const Tensor& x, const Tensor& z, const Tensor& scale, const Tensor& post_w, const Tensor& post_b,
                                              const Tensor& pre_w, const Tensor& pre_b, const std::optional<Tensor>& gate_, double eps) {
  const Tensor gate = gate_.value_or(Tensor());
  values_only("gated_norm_residual", {&x, &z, &scale, &post_w, &post_b, &pre_w, &pre_b, &gate});
  bool grads = false;
  for (const Tensor* t : {&x, &z, &scale, &post_w, &post_b, &pre_w, &pre_b, &gate}) grads = grads || (t->defined() && t->requires_grad());
  variable_list out;
  if (grads && at::GradMode::is_enabled()) {
    refuse_capture_beside_eager_graph("gated_norm_residual", {&x, &z, &scale, &post_w, &post_b, &pre_w, &pre_b, &gate});
    out = GatedNormResidual::apply(x, z, scale, post_w, post_b, pre_w, pre_b, gate_, eps);
  } else {
    const c10::DeviceGuard guard(x.device());
    const Tensor params[5] = {param(scale), param(post_w), param(post_b), param(pre_w), param(pre_b)};
    out = norm_forward(flat(x), flat(z), flat(gate), params, eps, nullptr);
  }
  return {out[0], out[1]};
}

}  // namespace

PYBIND11_MODULE(_atri_torch, m) {
  m.doc() = "Launch planning and autograd nodes of the encoder operators";
  m.def("bind", &bind);
  m.def("attention", &attention);
  m.def("gated_norm_residual", &gated_norm_residual);
}
