// torch's side of the operator in native code: argument checks, allocation, the autograd nodes of the operator, of the
// operator with group norm and gate and of the layer's input side, and the calls into libwkv6_gfx950.
//
// Why not Python: a training step is one or two kernel pairs of 40 to 110 us, and the same nodes written as
// torch.autograd.Function with ctypes calls took 185 us of host time per step at any size (265 with group norm and gate,
// 250 for the input side, 26 for one decoded token): every training shape up to about 2^25 elements ran at the speed of
// the interpreter, and the backward, which torch runs in a thread of its own, had to be handed the interpreter first.
//
// Rules of this file:
//  * every call holds no state between calls; tensors that outlive a forward are torch's saved variables (hooks and
//    version checks apply) or live in the node, as the saved chunk states do until the first backward takes them;
//  * `try_*` take a call only in its plain form and return None for anything else, and the Python layer then says what
//    is wrong with it or brings it into that form; what a call is refused for is decided there alone;
//  * kernels go to the current stream of the tensors' device; the interpreter's lock is not held meanwhile.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <initializer_list>
#include <optional>
#include <utility>
#include <vector>

#include "wkv6.h"

namespace {

namespace py = pybind11;
using at::ScalarType;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int kChunk = WKV6_ALGO_CHUNK;

int code_of(ScalarType t) {
  switch (t) {
    case at::kBFloat16: return WKV6_BF16;
    case at::kHalf: return WKV6_F16;
    case at::kFloat: return WKV6_F32;
    default: return -1;
  }
}

// rwkv_kernel/torch_rwkv_kernel.py:35 of the reference: float16 inputs produce float32 outputs
ScalarType out_type(ScalarType t) { return t == at::kHalf ? at::kFloat : t; }

// The package's own exception for a failed library call, also out of a backward's thread.
void check(int status) {
  if (status == 0) return;
  py::gil_scoped_acquire gil;
  try {
    py::module_::import("rwkv_kernel._native").attr("check")(status);
  } catch (py::error_already_set &e) {
    e.restore();
    python_error err;
    err.persist();
    throw err;
  }
}

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
// whether what goes to the current stream of the current device is recorded into a graph, to run any number of times
bool is_captured() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }

const void *in(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *out(const Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
const float *in_f(const Tensor &t) { return static_cast<const float *>(in(t)); }
float *out_f(const Tensor &t) { return static_cast<float *>(out(t)); }

Tensor bytes(const Tensor &like, size_t n) {
  return n ? at::empty({static_cast<int64_t>(n)}, at::TensorOptions().dtype(at::kByte).device(like.device())) : Tensor();
}

// Tensors of different shapes and types out of ONE allocation, each `slot` * 256 bytes past a 4 KiB boundary of it.  A
// workgroup of the kernels walks all (B,T,C) tensors of a call row by row in step; torch's allocator hands out large
// blocks on 2 MiB boundaries, and tensors whose bases agree modulo 4 KiB keep sending those streams to the same memory
// channel at the same moment (about 5 % of the training pair at B8 T1024 C2048).  The block lives as long as any of them.
struct Piece {
  at::DimVector shape;
  ScalarType type;
  int64_t slot;
};

std::vector<Tensor> carve(const Tensor &like, std::initializer_list<Piece> pieces) {
  std::vector<int64_t> offset;
  int64_t total = 0;
  for (const Piece &p : pieces) {
    const int64_t n = c10::multiply_integers(p.shape) * static_cast<int64_t>(c10::elementSize(p.type));
    offset.push_back(total + p.slot * 256);
    total += (p.slot * 256 + n + 4095) / 4096 * 4096;
  }
  const Tensor block = bytes(like, total ? total : 4096);
  std::vector<Tensor> res;
  size_t i = 0;
  for (const Piece &p : pieces) {
    auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(block.storage()), block.key_set(), c10::scalarTypeToTypeMeta(p.type));
    impl->set_storage_offset(offset[i++] / static_cast<int64_t>(c10::elementSize(p.type)));
    impl->set_sizes_contiguous(p.shape);
    res.emplace_back(std::move(impl));
  }
  return res;
}

// The gradient of a parameter gets an allocation of its own: torch takes it over as the parameter's .grad as it is, where it
// stays for as long as the caller keeps gradients, and with it whatever shares its block.
Tensor parameter_gradient(const Tensor &like, at::IntArrayRef shape, ScalarType type) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(like.device()));
}

bool any_requires_grad(std::initializer_list<const Tensor *> ts) {
  for (const Tensor *t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

struct Dims {
  int64_t B, T, C, H;
};

Dims dims_of(const Tensor &r, int64_t H) { return {r.size(0), r.size(1), r.size(2), H}; }

// The operator's backward from the arriving gradient: through the saved block when there is one, which it uses up.
// Gradients of r, k, v, w and u, in that order.
std::vector<Tensor> wkv6_grads(const Dims &d, int algo, const Tensor &r, const Tensor &k, const Tensor &v, const Tensor &w,
                               const Tensor &u, const Tensor &gy, const Tensor &saved) {
  const auto [B, T, C, H] = d;
  const int code = code_of(r.scalar_type());
  const ScalarType ot = out_type(r.scalar_type());
  const at::DimVector big{B, T, C};
  // torch hands the gradient of an fp16 tensor on as fp16 whatever a node returns, in a kernel per gradient: the library
  // rounds where it stores them, where its kernels can
  const ScalarType gt = saved.defined() && algo != kChunk ? r.scalar_type() : ot;
  std::vector<Tensor> g = carve(r, {{big, gt, 7}, {big, gt, 8}, {big, gt, 9}, {big, gt, 10}, {{B, C}, ot, 0}});
  const Tensor gu_rows = std::move(g[4]);
  if (saved.defined()) {
    g[4] = parameter_gradient(r, u.sizes(), gt);
    // the batch sum of u's gradient (rwkv_kernel/torch_rwkv_kernel.py:73 of the reference) comes out of the same launch
    check(wkv6_backward_saved_sum_ex(stream_of(r), code, code_of(gt), algo, B, T, C, H, in(r), in(k), in(v), in(w), in(u), in(gy),
                                     out(g[0]), out(g[1]), out(g[2]), out(g[3]), out(gu_rows), out(g[4]), out(saved), saved.numel()));
    return g;
  }
  const size_t n = wkv6_backward_workspace_bytes_ex(code, algo, B, T, C, H);
  const Tensor ws = bytes(r, n);
  check(wkv6_backward_ex(stream_of(r), code, algo, B, T, C, H, in(r), in(k), in(v), in(w), in(u), in(gy), out(g[0]), out(g[1]),
                         out(g[2]), out(g[3]), out(gu_rows), out(ws), n));
  g[4] = at::sum(gu_rows, 0).reshape(u.sizes());
  return g;
}

// The saved chunk states, handed from the forward to the first backward, which gives their memory back.  A second backward over
// the same graph (retain_graph) finds none and runs the plain backward.  (torch holds the node's lock while a backward runs.  One
// that is captured leaves the states as they were for its replays: each of them reads them and arms their counters again.)
// The same goes for sums that the forward cleared, which only one run of a backward can add to: see Wkv6GnGate.
void keep(AutogradContext *ctx, const Tensor &saved, const char *name = "states") {
  if (saved.defined()) ctx->saved_data[name] = saved;
}

Tensor take(AutogradContext *ctx, const char *name = "states") {
  auto it = ctx->saved_data.find(name);
  if (it == ctx->saved_data.end()) return Tensor();
  Tensor t = it->second.toTensor();
  ctx->saved_data.erase(it);
  return t;
}

// Stateless operator with gradients (rwkv_kernel/torch_rwkv_kernel.py:14-75 of the reference).  When a gradient will be
// needed and the library has something worth keeping for it (the chunked kernels' per-chunk states), the forward runs as
// wkv6_forward_save and the backward as wkv6_backward_saved_sum; otherwise the plain pair.
struct Wkv6 : torch::autograd::Function<Wkv6> {
  static Tensor forward(AutogradContext *ctx, const Tensor &r, const Tensor &k, const Tensor &v, const Tensor &w, const Tensor &u,
                        int64_t H, int64_t algo) {
    const c10::DeviceGuard guard(r.device());
    const auto [B, T, C, H_] = dims_of(r, H);
    const int code = code_of(r.scalar_type());
    const size_t nsave = any_requires_grad({&r, &k, &v, &w, &u}) ? wkv6_saved_bytes(code, algo, B, T, C, H) : 0;
    const Piece yp{{B, T, C}, out_type(r.scalar_type()), 5};
    Tensor y;
    if (nsave) {
      const auto t = carve(r, {yp, {{static_cast<int64_t>(nsave)}, at::kByte, 6}});
      y = t[0];
      check(wkv6_forward_save(stream_of(r), code, algo, B, T, C, H, in(r), in(k), in(v), in(w), in(u), out(y), out(t[1]), nsave));
      keep(ctx, t[1]);
    } else {
      y = carve(r, {yp})[0];
      // optional workspace: a long sequence of few (batch, head) pairs runs as time segments
      const size_t n = wkv6_forward_workspace_bytes_any_length(code, algo, B, T, C, H);
      const Tensor ws = bytes(r, n);
      // (no gradient is wanted, or the per-timestep kernels run, which read their inputs in one way only)
      check(wkv6_forward_inference(stream_of(r), code, code_of(out_type(r.scalar_type())), algo, B, T, C, H, 0, nullptr, in(r), in(k), in(v),
                                   in(w), in(u), nullptr, out(y), nullptr, out(ws), n));
    }
    ctx->saved_data["H"] = H;
    ctx->saved_data["algo"] = algo;
    ctx->save_for_backward({r, k, v, w, u});
    return y;
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const at::NoGradGuard no_grad;
    const auto s = ctx->get_saved_variables();
    const Tensor &r = s[0];
    const c10::DeviceGuard guard(r.device());
    TORCH_CHECK(grads[0].is_cuda() && grads[0].scalar_type() == out_type(r.scalar_type()), "wkv6: the gradient must have y's device and dtype");
    const Tensor gy = grads[0].contiguous();
    auto g = wkv6_grads(dims_of(r, ctx->saved_data["H"].toInt()), static_cast<int>(ctx->saved_data["algo"].toInt()), r, s[1], s[2],
                        s[3], s[4], gy, take(ctx));
    return {g[0], g[1], g[2], g[3], g[4], Tensor(), Tensor()};
  }
};

// out = (group_norm_head(wkv6(r, k, v, w, u)) * scale + offset) * gate, bf16, zero initial state: the operator and what the
// layer does with its output next (rwkv6_model.py:94-99,158-160 of the reference) in one forward kernel, the norm's and
// the gate's backward in one elementwise kernel, then the operator's backward from the saved chunk states.
struct Wkv6GnGate : torch::autograd::Function<Wkv6GnGate> {
  static Tensor forward(AutogradContext *ctx, const Tensor &r, const Tensor &k, const Tensor &v, const Tensor &w, const Tensor &u,
                        const Tensor &gate, const Tensor &scale, const Tensor &offset, int64_t H, double eps) {
    const c10::DeviceGuard guard(r.device());
    const auto [B, T, C, H_] = dims_of(r, H);
    const int code = code_of(r.scalar_type());
    const Tensor sc = scale.to(at::kFloat).contiguous(), of = offset.to(at::kFloat).contiguous();
    const int64_t nsave = wkv6_saved_bytes(code, kChunk, B, T, C, H);
    // out and what stays for the backward lie in blocks of their own: an output that a caller keeps holds nothing else
    const Tensor res = carve(r, {{{B, T, C}, r.scalar_type(), 5}})[0];
    const auto t = carve(r, {{{B, T, C}, r.scalar_type(), 6}, {{nsave}, at::kByte, 7}, {{B, T, H, 2}, at::kFloat, 0}});
    if (is_captured()) {   // (each replay would clear the sums again, and with them the gradients a backward gave out)
      check(wkv6_forward_gn_gate_save(stream_of(r), code, B, T, C, H, in(r), in(k), in(v), in(w), in(u), in(gate), in_f(sc), in_f(of),
                                      static_cast<float>(eps), out(res), out(t[0]), out_f(t[2]), out(t[1]), nsave));
    } else {
      // the norm's gradients, which this forward clears for the first backward to add to
      const Tensor gscale = parameter_gradient(r, sc.sizes(), at::kFloat), goffset = parameter_gradient(r, of.sizes(), at::kFloat);
      check(wkv6_forward_gn_gate_save_sums(stream_of(r), code, B, T, C, H, in(r), in(k), in(v), in(w), in(u), in(gate), in_f(sc), in_f(of),
                                           static_cast<float>(eps), out(res), out(t[0]), out_f(t[2]), out(t[1]), nsave, out_f(gscale),
                                           out_f(goffset)));
      keep(ctx, gscale, "gscale");
      keep(ctx, goffset, "goffset");
    }
    keep(ctx, t[1]);
    ctx->saved_data["H"] = H;
    ctx->saved_data["scale_type"] = static_cast<int64_t>(scale.scalar_type());
    ctx->saved_data["offset_type"] = static_cast<int64_t>(offset.scalar_type());
    ctx->save_for_backward({r, k, v, w, u, gate, sc, of, t[0], t[2]});
    return res;
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const at::NoGradGuard no_grad;
    const auto s = ctx->get_saved_variables();
    const Tensor &r = s[0];
    const c10::DeviceGuard guard(r.device());
    const Dims d = dims_of(r, ctx->saved_data["H"].toInt());
    const auto [B, T, C, H] = d;
    TORCH_CHECK(grads[0].scalar_type() == r.scalar_type(), "wkv6: the gradient must have the output's dtype");
    const Tensor gout = grads[0].contiguous();
    const ScalarType t = r.scalar_type();
    const Tensor gy = carve(r, {{{B, T, C}, t, 5}})[0];
    const Tensor ggate = carve(r, {{{B, T, C}, t, 6}})[0];
    // (captured: the forward cleared its sums once, while the replays of this backward, however many follow one forward, each have to
    // start from zero, in memory of the graph's own)
    Tensor gscale, goffset;
    if (!is_captured()) { gscale = take(ctx, "gscale"); goffset = take(ctx, "goffset"); }
    const auto norm_backward = gscale.defined() ? wkv6_gn_gate_backward_sums : wkv6_gn_gate_backward;
    if (!gscale.defined()) {   // (also a second backward over the same graph, and one whose forward was captured)
      gscale = parameter_gradient(r, s[6].sizes(), at::kFloat);
      goffset = parameter_gradient(r, s[7].sizes(), at::kFloat);
    }
    check(norm_backward(stream_of(r), code_of(t), B, T, C, H, in(gout), in(s[8]), in_f(s[9]), in(s[5]), in_f(s[6]), in_f(s[7]), out(gy),
                        out(ggate), out_f(gscale), out_f(goffset)));
    auto w = wkv6_grads(d, kChunk, r, s[1], s[2], s[3], s[4], gy, take(ctx));
    return {w[0], w[1], w[2], w[3], w[4], ggate,
            gscale.to(static_cast<ScalarType>(ctx->saved_data["scale_type"].toInt())),
            goffset.to(static_cast<ScalarType>(ctx->saved_data["offset_type"].toInt())), Tensor(), Tensor()};
  }
};

// A parameter as the kernels read it: of this type, contiguous and on a 16-byte boundary.  (One that already has the type and
// is contiguous may be a view into a flat buffer of parameters, anywhere in it.)
Tensor laid_out(const Tensor &t, ScalarType type) {
  const Tensor c = t.to(type).contiguous();
  return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 == 0 ? c : c.clone();
}

// The layer's input side (rwkv6_model.py:134-146 of the reference) with gradients, bf16: x -> (xr, xk, xv, xw, xg).
struct ShiftMix : torch::autograd::Function<ShiftMix> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &mix_x, const Tensor &a, const Tensor &w2t,
                               const Tensor &bias) {
    const c10::DeviceGuard guard(x.device());
    const int64_t B = x.size(0), T = x.size(1), C = x.size(2), R = w2t.size(2);
    const int code = code_of(x.scalar_type());
    const Tensor mx = mix_x.to(at::kFloat).contiguous(), b32 = bias.to(at::kFloat).contiguous();
    const ScalarType wt = a.scalar_type() == w2t.scalar_type() && a.scalar_type() == at::kBFloat16 ? at::kBFloat16 : at::kFloat;
    // (bf16 second weights are handed through, and refused off a 16-byte boundary, like x and the biases)
    const Tensor aw = laid_out(a, wt), ww = w2t.scalar_type() == at::kBFloat16 ? w2t.to(wt).contiguous() : laid_out(w2t, wt);
    const int64_t nw = wkv6_shift_mix_weights_bytes(C, R);
    const ScalarType t = x.scalar_type();
    const at::DimVector big{B, T, C};
    auto o = carve(x, {{big, t, 1}, {big, t, 2}, {big, t, 3}, {big, t, 4}, {big, t, 5}});
    // (not out of the outputs' block: a caller may change an output in place)
    const auto kept = carve(x, {{{B, T, 5 * R}, t, 6}, {{nw}, at::kByte, 0}});
    check(wkv6_shift_mix_forward(stream_of(x), code, code_of(wt), B, T, C, R, in(x), in_f(mx), in(aw), in(ww), in_f(b32), out(kept[1]),
                                 nw, out(kept[0]), out(o[0]), out(o[1]), out(o[2]), out(o[3]), out(o[4])));
    ctx->saved_data["weight_type"] = static_cast<int64_t>(wt);
    ctx->saved_data["types"] = std::vector<int64_t>{static_cast<int64_t>(mix_x.scalar_type()), static_cast<int64_t>(a.scalar_type()),
                                                    static_cast<int64_t>(w2t.scalar_type()), static_cast<int64_t>(bias.scalar_type())};
    ctx->save_for_backward({x, kept[0], kept[1], mx, b32});
    return o;
  }

  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const at::NoGradGuard no_grad;
    const auto s = ctx->get_saved_variables();
    const Tensor &x = s[0], &h = s[1], &weights = s[2], &mx = s[3], &b32 = s[4];
    const c10::DeviceGuard guard(x.device());
    const int64_t B = x.size(0), T = x.size(1), C = x.size(2), R = h.size(2) / 5;
    const ScalarType t = x.scalar_type(), wt = static_cast<ScalarType>(ctx->saved_data["weight_type"].toInt());
    const int code = code_of(t);
    for (Tensor &g : grads) g = g.to(t).contiguous();
    const Tensor gx = carve(x, {{{B, T, C}, t, 6}})[0];
    const Tensor gmix = parameter_gradient(x, {C}, at::kFloat), ga = parameter_gradient(x, {5 * R, C}, wt),
                 gw2t = parameter_gradient(x, {5, C, R}, wt), gbias = parameter_gradient(x, {5, C}, at::kFloat);
    const size_t n = wkv6_shift_mix_backward_workspace_bytes(code, B, T, C, R);
    const Tensor ws = bytes(x, n);
    check(wkv6_shift_mix_backward(stream_of(x), code, code_of(wt), B, T, C, R, in(x), in_f(mx), in_f(b32), in(weights), in(h),
                                  in(grads[0]), in(grads[1]), in(grads[2]), in(grads[3]), in(grads[4]), out(gx), out_f(gmix),
                                  out(ga), out(gw2t), out_f(gbias), out(ws), n));
    const auto types = ctx->saved_data["types"].toIntVector();
    const auto as = [&](const Tensor &v, int i) { return v.to(static_cast<ScalarType>(types[i])); };
    return {gx, as(gmix, 0), as(ga, 1), as(gw2t, 2), as(gbias, 3)};
  }
};

// ---- losses over logits (wkv6_token_logprobs and its kin) ----

// Logits as the kernels read them: (B, T, V), a row's values next to each other.
struct Logits {
  Tensor x, ids, mask;
  int64_t B, T, V;
  int code;
  const int64_t *id() const { return static_cast<const int64_t *>(in(ids)); }
  const uint8_t *counted() const { return static_cast<const uint8_t *>(in(mask)); }
};

Tensor given(const std::optional<Tensor> &t) { return t.has_value() ? *t : Tensor(); }

Logits logits_of(const Tensor &x, const Tensor &ids, const std::optional<Tensor> &mask) {
  return {x, ids, given(mask), x.size(0), x.size(1), x.size(2), code_of(x.scalar_type())};
}

Tensor fp32(const Tensor &like, at::IntArrayRef shape) { return at::empty(shape, like.options().dtype(at::kFloat)); }

// What a node keeps of the rows for its backward.
void keep_rows(AutogradContext *ctx, const Logits &l, const Tensor &stats, const Tensor &coef, double temperature) {
  ctx->saved_data["temperature"] = temperature;
  ctx->save_for_backward({l.x, l.ids, l.mask, stats, coef});
}

// Memory for the gradient that a forward writes beside its loss, or nothing where the backward writes it: in half precision, where
// a training scales its loss up for the gradient's sake (so what arrives is not 1, and what is too small without it would be
// lost here), and into a graph, whose replays may run the backward again and again after one forward.
Tensor gradient_ahead(const Logits &l, bool wanted) {
  if (!wanted || l.x.scalar_type() == at::kHalf || is_captured()) return Tensor();
  return at::empty({l.B, l.T, l.V}, l.x.options());
}

// The gradient by the logits of sum(coef * logps), times `upstream` (undefined for 1).  `ahead`: what a forward wrote, for an upstream of 1.
Tensor logits_backward(const variable_list &saved, double temperature, const Tensor &coef, int64_t coef_stride_b, int64_t coef_stride_t,
                       const Tensor &upstream, const Tensor &ahead) {
  const Logits l = logits_of(saved[0], saved[1], saved[2]);
  const Tensor grad = ahead.defined() ? ahead : at::empty({l.B, l.T, l.V}, l.x.options());
  check(wkv6_logits_backward(stream_of(l.x), l.code, l.B, l.T, l.V, in(l.x), l.x.stride(0), l.x.stride(1), l.id(), l.counted(),
                             static_cast<float>(temperature), in_f(saved[3]), in_f(coef), coef_stride_b, coef_stride_t, in_f(upstream),
                             ahead.defined(), out(grad)));
  return grad;
}

Tensor arriving(const Tensor &g) { return g.to(at::kFloat).contiguous(); }

// Stands for what a gradient depends on where a graph of the backward is wanted (create_graph): the gradient has its value, and a derivative of it
// is refused, where without a node it would be missing from whatever it is a part of.
struct FirstOrder : torch::autograd::Function<FirstOrder> {
  static Tensor forward(AutogradContext *, const Tensor &grad, const Tensor &, const Tensor &) { return grad; }
  static variable_list backward(AutogradContext *, variable_list) {
    TORCH_CHECK(false, "wkv6: the losses over logits have no second derivative");
  }
};

Tensor first_order(bool graph_wanted, const Tensor &grad, const Tensor &logits, const Tensor &arrived) {
  if (!graph_wanted) return grad;
  const at::AutoGradMode on(true);
  return FirstOrder::apply(grad, logits, arrived);
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &ids, const std::optional<Tensor> &mask, double temperature, bool wanted) {
    const c10::DeviceGuard guard(x.device());
    const Logits l = logits_of(x, ids, mask);
    const Tensor lp = fp32(x, {l.B, l.T}), stats = wanted ? fp32(x, {l.B, l.T, 2}) : Tensor();
    check(wkv6_token_logprobs(stream_of(x), l.code, l.B, l.T, l.V, in(x), x.stride(0), x.stride(1), l.id(), l.counted(),
                              static_cast<float>(temperature), out_f(lp), out_f(stats)));
    keep_rows(ctx, l, stats, Tensor(), temperature);
    return lp;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const bool graph_wanted = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    const auto s = ctx->get_saved_variables();
    const c10::DeviceGuard guard(s[0].device());
    const Tensor coef = arriving(grads[0]);
    const Tensor grad = logits_backward(s, ctx->saved_data["temperature"].toDouble(), coef, s[0].size(1), 1, Tensor(), Tensor());
    return {first_order(graph_wanted, grad, s[0], grads[0]), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct CrossEntropy : torch::autograd::Function<CrossEntropy> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &ids, const std::optional<Tensor> &mask, int64_t reduction, bool wanted) {
    const c10::DeviceGuard guard(x.device());
    const Logits l = logits_of(x, ids, mask);
    const Tensor loss = fp32(x, {}), stats = wanted ? fp32(x, {l.B, l.T, 2}) : Tensor(), coef = wanted ? fp32(x, {l.B, l.T}) : Tensor();
    const Tensor grad = gradient_ahead(l, wanted);
    const size_t n = wkv6_loss_workspace_bytes(l.B, l.T);
    const Tensor ws = bytes(x, n);
    check(wkv6_cross_entropy(stream_of(x), l.code, l.B, l.T, l.V, in(x), x.stride(0), x.stride(1), l.id(), l.counted(),
                             static_cast<int>(reduction), out_f(loss), out_f(stats), out_f(coef), out(grad), out(ws), n));
    keep_rows(ctx, l, stats, coef, 1.0);
    keep(ctx, grad, "grad");
    return loss;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const bool graph_wanted = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    const auto s = ctx->get_saved_variables();
    const c10::DeviceGuard guard(s[0].device());
    const Tensor ahead = is_captured() ? Tensor() : take(ctx, "grad"), up = arriving(grads[0]);
    const Tensor grad = logits_backward(s, ctx->saved_data["temperature"].toDouble(), s[4], s[0].size(1), 1, up, ahead);
    return {first_order(graph_wanted, grad, s[0], grads[0]), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &ids, const std::optional<Tensor> &mask, const std::optional<Tensor> &old_logps,
                               const Tensor &advantages, const std::optional<Tensor> &ref_logps, double clip_low, double clip_high, double kl_weight,
                               double temperature, int64_t reduction, bool wanted) {
    const c10::DeviceGuard guard(x.device());
    const Logits l = logits_of(x, ids, mask);
    const Tensor loss = fp32(x, {}), lp = fp32(x, {l.B, l.T}), means = fp32(x, {2});
    const Tensor stats = wanted ? fp32(x, {l.B, l.T, 2}) : Tensor(), coef = wanted ? fp32(x, {l.B, l.T}) : Tensor();
    const Tensor grad = gradient_ahead(l, wanted);
    const size_t n = wkv6_loss_workspace_bytes(l.B, l.T);
    const Tensor ws = bytes(x, n);
    check(wkv6_policy_loss(stream_of(x), l.code, l.B, l.T, l.V, in(x), x.stride(0), x.stride(1), l.id(), l.counted(), in_f(given(old_logps)),
                           in_f(advantages), advantages.stride(0), advantages.dim() == 2 ? advantages.stride(1) : 0, in_f(given(ref_logps)), static_cast<float>(clip_low),
                           static_cast<float>(clip_high), static_cast<float>(kl_weight), static_cast<float>(temperature),
                           static_cast<int>(reduction), out_f(loss), out_f(lp), out_f(means), out_f(stats), out_f(coef), out(grad), out(ws), n));
    keep_rows(ctx, l, stats, coef, temperature);
    keep(ctx, grad, "grad");
    ctx->mark_non_differentiable({lp, means});
    ctx->set_materialize_grads(false);
    return {loss, lp, means};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const bool graph_wanted = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    variable_list res(12);
    if (!grads[0].defined()) return res;
    const auto s = ctx->get_saved_variables();
    const c10::DeviceGuard guard(s[0].device());
    const Tensor ahead = is_captured() ? Tensor() : take(ctx, "grad"), up = arriving(grads[0]);
    res[0] = first_order(graph_wanted, logits_backward(s, ctx->saved_data["temperature"].toDouble(), s[4], s[0].size(1), 1, up, ahead), s[0], grads[0]);
    return res;
  }
};

struct PreferenceLoss : torch::autograd::Function<PreferenceLoss> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &ids, const std::optional<Tensor> &mask, const std::optional<Tensor> &ref_logps,
                               int64_t kind, double beta, double label_smoothing, bool average, bool wanted) {
    const c10::DeviceGuard guard(x.device());
    const Logits l = logits_of(x, ids, mask);
    const Tensor loss = fp32(x, {}), text = fp32(x, {l.B});
    const Tensor stats = wanted ? fp32(x, {l.B, l.T, 2}) : Tensor(), coef = wanted ? fp32(x, {l.B}) : Tensor();
    const size_t n = wkv6_loss_workspace_bytes(l.B, l.T);
    const Tensor ws = bytes(x, n);
    check(wkv6_preference_loss(stream_of(x), l.code, l.B, l.T, l.V, in(x), x.stride(0), x.stride(1), l.id(), l.counted(), in_f(given(ref_logps)),
                               static_cast<int>(kind), beta, label_smoothing, average, out_f(loss), out_f(text), out_f(stats), out_f(coef), out(ws), n));
    keep_rows(ctx, l, stats, coef, 1.0);
    ctx->mark_non_differentiable({text});
    ctx->set_materialize_grads(false);
    return {loss, text};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const bool graph_wanted = at::GradMode::is_enabled();
    const at::NoGradGuard no_grad;
    variable_list res(9);
    if (!grads[0].defined()) return res;
    const auto s = ctx->get_saved_variables();
    const c10::DeviceGuard guard(s[0].device());
    res[0] = first_order(graph_wanted, logits_backward(s, 1.0, s[4], 1, 0, arriving(grads[0]), Tensor()), s[0], grads[0]);
    return res;
  }
};

// ---- AdamW ----

bool same_layout(const Tensor &a, const Tensor &b) {
  return a.sizes() == b.sizes() && (a.strides() == b.strides() || (a.is_contiguous() && b.is_contiguous()));
}

using Tensors = std::vector<Tensor>;

void on_one_device(const Tensor &t, const Tensor &like, const char *what) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), "wkv6: ", what, " must be on the parameters' GPU");
}

Tensor grad_norm(const Tensors &grads) {
  TORCH_CHECK(!grads.empty() && grads[0].is_cuda() && code_of(grads[0].scalar_type()) >= 0, "wkv6: gradients are bf16, fp16 or fp32 tensors on the GPU");
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(grads[0].device());
  Tensors kept;   // (dense copies of what is not, until the kernels are enqueued)
  std::vector<wkv6_adamw_tensor> rows;
  for (const Tensor &g : grads) {
    on_one_device(g, grads[0], "gradients");
    TORCH_CHECK(g.scalar_type() == grads[0].scalar_type() && g.layout() == at::kStrided, "wkv6: gradients are dense and of one dtype");
    const Tensor d = g.is_non_overlapping_and_dense() ? g : g.contiguous();
    kept.push_back(d);
    rows.push_back({nullptr, in(d), nullptr, nullptr, nullptr, nullptr, d.numel()});
  }
  const Tensor norm = fp32(grads[0], {});
  const size_t n = wkv6_grad_norm_workspace_bytes(rows.size());
  const Tensor ws = bytes(grads[0], n);
  check(wkv6_grad_norm(stream_of(grads[0]), code_of(grads[0].scalar_type()), rows.size(), rows.data(), out_f(norm), out(ws), n));
  return norm;
}

// The step; returns the gradients' norm, `norm` itself where it is given, nothing where nobody asks for it.
Tensor adamw_step(const Tensors &params, const Tensors &grads, const Tensors &exp_avgs, const Tensors &exp_avg_sqs, const Tensor &step,
                  const Tensors &scales, const Tensors &masters, const Tensor &lr_device, double lr, double beta1, double beta2, double eps,
                  double weight_decay, double max_grad_norm, bool skip_nonfinite, Tensor norm, int64_t seed) {
  const size_t count = params.size();
  TORCH_CHECK(count > 0 && grads.size() == count && exp_avgs.size() == count && exp_avg_sqs.size() == count,
              "wkv6: one gradient and two moments for each parameter");
  const Tensor &first = params[0];
  const ScalarType type = first.scalar_type(), moment = exp_avgs[0].scalar_type();
  TORCH_CHECK(first.is_cuda() && code_of(type) >= 0, "wkv6: parameters are bf16, fp16 or fp32 tensors on the GPU");
  TORCH_CHECK(moment == at::kFloat || moment == at::kFloat8_e4m3fn, "wkv6: moments are float32 or float8_e4m3fn");
  const bool eight = moment == at::kFloat8_e4m3fn;
  TORCH_CHECK(eight ? scales.size() == count : scales.empty(), "wkv6: moments in 8 bits, and no others, have scales");
  TORCH_CHECK(masters.empty() || (masters.size() == count && type != at::kFloat), "wkv6: one master for each parameter of 16 bits");
  on_one_device(step, first, "step");
  TORCH_CHECK(step.scalar_type() == at::kLong && step.numel() == 1, "wkv6: step is one int64");
  for (const Tensor *t : {&lr_device, const_cast<const Tensor *>(&norm)}) {
    if (!t->defined()) continue;
    on_one_device(*t, first, "lr and grad_norm");
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->numel() == 1, "wkv6: lr and grad_norm are one float32");
  }
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(first.device());
  Tensors kept;
  std::vector<wkv6_adamw_tensor> rows;
  std::vector<std::pair<uintptr_t, uintptr_t>> seen;   // what is written, from and to
  for (size_t i = 0; i < count; ++i) {
    const Tensor &p = params[i], &m = exp_avgs[i], &v = exp_avg_sqs[i];
    for (const Tensor *t : {&p, &grads[i], &m, &v}) {
      on_one_device(*t, first, "gradients and moments");
      TORCH_CHECK(t->layout() == at::kStrided && t->sizes() == p.sizes(), "wkv6: a gradient and its moments have the parameter's shape");
    }
    TORCH_CHECK(p.scalar_type() == type && grads[i].scalar_type() == type, "wkv6: parameters and gradients of a call have one dtype");
    TORCH_CHECK(m.scalar_type() == moment && v.scalar_type() == moment, "wkv6: moments of a call have one dtype");
    TORCH_CHECK(p.is_non_overlapping_and_dense() && same_layout(m, p) && same_layout(v, p), "wkv6: parameters are dense, their moments laid out like them");
    wkv6_adamw_tensor row{out(p), nullptr, out(m), out(v), nullptr, nullptr, p.numel()};
    if (eight) {
      on_one_device(scales[i], first, "scales");
      TORCH_CHECK(scales[i].scalar_type() == at::kFloat && scales[i].is_contiguous() && scales[i].dim() == 2 && scales[i].size(1) == 2 &&
                      scales[i].size(0) == (p.numel() + 255) / 256, "wkv6: scales are float32 (ceil(numel / 256), 2)");
      row.scales = out_f(scales[i]);
    }
    if (!masters.empty()) {
      on_one_device(masters[i], first, "masters");
      TORCH_CHECK(masters[i].scalar_type() == at::kFloat && same_layout(masters[i], p), "wkv6: masters are float32, laid out like their parameters");
      row.master = out_f(masters[i]);
    }
    Tensor g = grads[i];
    if (!same_layout(g, p)) g = at::empty_like(p).copy_(g);
    kept.push_back(g);
    row.grad = in(g);
    rows.push_back(row);
    const int64_t n = p.numel(), moment_bytes = n * (eight ? 1 : 4);
    for (const auto &[written, size] : {std::pair<void *, int64_t>{row.param, n * p.element_size()}, {row.exp_avg, moment_bytes}, {row.exp_avg_sq, moment_bytes},
                                        {row.scales, (n + 255) / 256 * 8}, {row.master, n * 4}})
      if (written && n > 0) seen.emplace_back(reinterpret_cast<uintptr_t>(written), reinterpret_cast<uintptr_t>(written) + size);
  }
  // (in order of where they begin, one that reaches into another reaches into the next)
  std::sort(seen.begin(), seen.end());
  for (size_t i = 1; i < seen.size(); ++i)
    TORCH_CHECK(seen[i - 1].second <= seen[i].first, "wkv6: a parameter, a moment, its scales or a master is given twice, or shares elements with another");
  if (!norm.defined() && (max_grad_norm > 0. || skip_nonfinite)) norm = grad_norm(kept);
  check(wkv6_adamw_step(stream_of(first), code_of(type), eight ? 8 : 32, count, rows.data(), static_cast<int64_t *>(out(step)), in_f(lr_device), lr, beta1,
                        beta2, eps, weight_decay, max_grad_norm, skip_nonfinite, in_f(norm), static_cast<uint32_t>(seed)));
  for (const Tensors *l : {&params, &exp_avgs, &exp_avg_sqs, &scales, &masters})
    for (const Tensor &t : *l)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();   // (what autograd saved of them is no longer what it was)
  if (!step.is_inference()) step.unsafeGetTensorImpl()->bump_version();
  return norm;
}

// (B, H, N, N)
at::DimVector state_shape(const Dims &d) {
  TORCH_CHECK(d.H > 0, "wkv6: tensors without channels have no state");   // (the size per head below divides by it)
  return {d.B, d.H, d.C / d.H, d.C / d.H};
}

// Stateful forward without a gradient (rwkv_kernel/torch_rwkv_kernel.py:76-95 of the reference): y and the final state.
// An undefined map with an initial state means row b starts from s0[b].
std::pair<Tensor, Tensor> forward_with_state(int64_t H, const Tensor &map, const Tensor &r, const Tensor &k, const Tensor &v,
                                             const Tensor &w, const Tensor &u, const Tensor &s0, int64_t algo, ScalarType st,
                                             bool backward_follows = false) {
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(r.device());
  const Dims d = dims_of(r, H);
  const auto [B, T, C, H_] = d;
  const int code = code_of(r.scalar_type());
  const Tensor y = carve(r, {{{B, T, C}, out_type(r.scalar_type()), 5}})[0];
  const Tensor ys = at::empty(state_shape(d), r.options().dtype(st));
  // optional workspace: a long sequence of few (batch, head) pairs runs as time segments
  const size_t n = wkv6_forward_workspace_bytes_any_length(code, algo, B, T, C, H);
  const Tensor ws = bytes(r, n);
  const auto forward = backward_follows ? wkv6_forward_with_state_ex : wkv6_forward_inference;
  check(forward(stream_of(r), code, code_of(st), algo, B, T, C, H, s0.defined(), static_cast<const int64_t *>(in(map)), in(r), in(k),
                in(v), in(w), in(u), in(s0), out(y), out(ys), out(ws), n));
  return {y, ys};
}

// The same with group norm and gate in the output stage; the final state only on request.
std::pair<Tensor, Tensor> forward_gn_gate(int64_t H, const Tensor &map, const Tensor &r, const Tensor &k, const Tensor &v,
                                          const Tensor &w, const Tensor &u, const Tensor &s0, const Tensor &gate, const Tensor &scale,
                                          const Tensor &offset, double eps, bool want_state) {
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(r.device());
  const Dims d = dims_of(r, H);
  const auto [B, T, C, H_] = d;
  const int code = code_of(r.scalar_type());
  const Tensor sc = scale.to(r.device(), at::kFloat).contiguous(), of = offset.to(r.device(), at::kFloat).contiguous();
  const ScalarType st = s0.defined() ? s0.scalar_type() : at::kFloat;
  const Tensor res = carve(r, {{{B, T, C}, r.scalar_type(), 5}})[0];
  const Tensor ys = want_state ? at::empty(state_shape(d), r.options().dtype(st)) : Tensor();
  const size_t n = wkv6_forward_workspace_bytes_any_length(code, kChunk, B, T, C, H);
  const Tensor ws = bytes(r, n);
  check(wkv6_forward_gn_gate_ex(stream_of(r), code, code_of(st), B, T, C, H, s0.defined(), static_cast<const int64_t *>(in(map)), in(r),
                                in(k), in(v), in(w), in(u), in(s0), in(gate), in_f(sc), in_f(of), static_cast<float>(eps), out(res),
                                out(ys), out(ws), n));
  return {res, ys};
}

// A tensor that takes no part in a graph.
Tensor apart(const Tensor &t) { return t.defined() && t.requires_grad() ? t.detach() : t; }
std::optional<Tensor> apart(const std::optional<Tensor> &t) { return t.has_value() ? std::optional<Tensor>(apart(*t)) : t; }

// ---- what the Python layer calls ----

// r, k, v, w and u as the kernels take them, with nothing left for the Python layer to check or to change.
bool plain(int64_t N, const Tensor &r, const Tensor &k, const Tensor &v, const Tensor &w, const Tensor &u) {
  if (r.dim() != 3 || !r.is_cuda() || code_of(r.scalar_type()) < 0 || r.size(2) == 0 || r.size(2) % N != 0 || u.numel() != r.size(2))
    return false;
  for (const Tensor *t : {&r, &k, &v, &w, &u})
    if (t->device() != r.device() || t->scalar_type() != r.scalar_type() || !t->is_contiguous()) return false;
  return k.sizes() == r.sizes() && v.sizes() == r.sizes() && w.sizes() == r.sizes();
}

// An initial state as the kernels take it, one per batch row.
bool plain_state(int64_t N, const Tensor &r, const Tensor &s) {
  return s.dim() == 4 && s.size(0) == r.size(0) && s.size(1) == r.size(2) / N && s.size(2) == N && s.size(3) == N &&
         s.device() == r.device() && s.is_contiguous() && (s.scalar_type() == at::kFloat || s.scalar_type() == out_type(r.scalar_type()));
}

const Tensor *tensor(const py::object &o) { return THPVariable_Check(o.ptr()) ? &THPVariable_Unpack(o.ptr()) : nullptr; }

py::object wrap(const Tensor &t) { return t.defined() ? py::reinterpret_steal<py::object>(THPVariable_Wrap(t)) : py::none(); }

// Whatever Python takes for true or false (pybind11's bool refuses lists, texts and other objects with a length).
bool truth(const py::object &o) {
  const int t = PyObject_IsTrue(o.ptr());
  if (t < 0) throw py::error_already_set();
  return t != 0;
}

py::tuple wrap(const std::pair<Tensor, Tensor> &p) { return py::make_tuple(wrap(p.first), wrap(p.second)); }

// Runs f without the interpreter's lock.  A Python error that torch has put into a C++ exception is restored as it was.
template <typename F> auto unlocked(F &&f) {
  try {
    py::gil_scoped_release nogil;
    return f();
  } catch (python_error &e) {
    py::gil_scoped_acquire gil;
    e.restore();
    throw py::error_already_set();
  }
}

py::object try_call(int64_t N, int64_t algo, const py::object &r_, const py::object &k_, const py::object &v_, const py::object &w_,
                    const py::object &u_, const py::object &return_state_, const py::object &s0_) {
  const Tensor *r = tensor(r_), *k = tensor(k_), *v = tensor(v_), *w = tensor(w_), *u = tensor(u_), *s0 = tensor(s0_);
  if (!r || !k || !v || !w || !u || !plain(N, *r, *k, *v, *w, *u)) return py::none();
  const int64_t H = r->size(2) / N;
  if (!truth(return_state_)) {
    if (!s0_.is_none()) return py::none();
    return py::make_tuple(wrap(unlocked([&] { return Wkv6::apply(*r, *k, *v, *w, *u, H, algo); })), py::none());
  }
  const Tensor state = s0 ? *s0 : Tensor();
  if (s0 ? !plain_state(N, *r, state) : !s0_.is_none()) return py::none();
  if (at::GradMode::is_enabled() && any_requires_grad({r, k, v, w, u, &state})) return py::none();
  const ScalarType st = s0 ? state.scalar_type() : out_type(r->scalar_type());
  return wrap(unlocked([&] { return forward_with_state(H, Tensor(), *r, *k, *v, *w, *u, state, algo, st); }));
}

py::object try_gn_gate(int64_t N, const py::object &r_, const py::object &k_, const py::object &v_, const py::object &w_,
                       const py::object &u_, const py::object &gate_, const py::object &scale_, const py::object &offset_,
                       const py::object &eps_, const py::object &return_state_, const py::object &s0_) {
  const Tensor *r = tensor(r_), *k = tensor(k_), *v = tensor(v_), *w = tensor(w_), *u = tensor(u_), *s0 = tensor(s0_);
  const Tensor *gate = tensor(gate_), *scale = tensor(scale_), *offset = tensor(offset_);
  if (!r || !k || !v || !w || !u || !gate || !scale || !offset || !plain(N, *r, *k, *v, *w, *u)) return py::none();
  const int64_t B = r->size(0), T = r->size(1), C = r->size(2), H = C / N;
  if (r->scalar_type() != at::kBFloat16 || gate->sizes() != r->sizes() || gate->scalar_type() != r->scalar_type() ||
      gate->device() != r->device() || !gate->is_contiguous() || scale->numel() != C || offset->numel() != C ||
      scale->device() != r->device() || offset->device() != r->device())
    return py::none();
  const Tensor state = s0 ? *s0 : Tensor();
  if (s0 ? !plain_state(N, *r, state) : !s0_.is_none()) return py::none();
  const bool return_state = truth(return_state_);
  const double eps = py::float_(eps_);
  if (at::GradMode::is_enabled() && any_requires_grad({r, k, v, w, u, gate, scale, offset})) {
    if (return_state || s0 || !wkv6_forward_gn_gate_save_supported(code_of(r->scalar_type()), B, T, C, H)) return py::none();
    return py::make_tuple(wrap(unlocked([&] { return Wkv6GnGate::apply(*r, *k, *v, *w, *u, *gate, *scale, *offset, H, eps); })), py::none());
  }
  return wrap(unlocked([&] {
    return forward_gn_gate(H, Tensor(), *r, *k, *v, *w, *u, state, *gate, *scale, *offset, eps, return_state);
  }));
}

}  // namespace

PYBIND11_MODULE(_wkv6_torch, m) {
  m.def("try_call", &try_call);
  m.def("try_gn_gate", &try_gn_gate);
  m.def("wkv6", [](const Tensor &r, const Tensor &k, const Tensor &v, const Tensor &w, const Tensor &u, int64_t H, int64_t algo) {
    return unlocked([&] { return Wkv6::apply(r, k, v, w, u, H, algo); });
  });
  m.def("wkv6_gn_gate", [](const Tensor &r, const Tensor &k, const Tensor &v, const Tensor &w, const Tensor &u, const Tensor &gate,
                           const Tensor &scale, const Tensor &offset, int64_t H, double eps) {
    return unlocked([&] { return Wkv6GnGate::apply(r, k, v, w, u, gate, scale, offset, H, eps); });
  });
  m.def("shift_mix", [](const Tensor &x, const Tensor &mix_x, const Tensor &a, const Tensor &w2t, const Tensor &bias) {
    for (const Tensor *t : {&mix_x, &a, &w2t, &bias})
      TORCH_CHECK(t->device() == x.device(), "wkv6: x and the mixers' parameters must be on one device");   // (the kernels take addresses)
    const variable_list o = unlocked([&] { return ShiftMix::apply(x, mix_x, a, w2t, bias); });
    return py::make_tuple(wrap(o[0]), wrap(o[1]), wrap(o[2]), wrap(o[3]), wrap(o[4]));
  });
  m.def("forward_with_state", [](int64_t H, const std::optional<Tensor> &map, const Tensor &r, const Tensor &k, const Tensor &v,
                                 const Tensor &w, const Tensor &u, const std::optional<Tensor> &s0, int64_t algo, int state_code,
                                 bool backward_follows) {
    const ScalarType st = state_code == WKV6_F32 ? at::kFloat : state_code == WKV6_F16 ? at::kHalf : at::kBFloat16;
    return wrap(unlocked([&] { return forward_with_state(H, given(map), r, k, v, w, u, given(s0), algo, st, backward_follows); }));
  }, py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg(), py::arg("backward_follows") = false);
  // Logits, ids and a mask (or None) as the kernels take them, with nothing left for the Python layer to check or to change.
  m.def("plain_rows", [](const py::object &x_, const py::object &ids_, const py::object &mask_) {
    const Tensor *x = tensor(x_), *ids = tensor(ids_), *mask = tensor(mask_);
    if (!x || !ids || !(mask || mask_.is_none()) || !x->is_cuda() || x->dim() != 3 || code_of(x->scalar_type()) < 0 || x->size(2) == 0 || x->stride(2) != 1)
      return false;
    const auto beside = [&](const Tensor &t) {
      return t.device() == x->device() && t.dim() == 2 && t.size(0) == x->size(0) && t.size(1) == x->size(1) && t.is_contiguous();
    };
    return ids->scalar_type() == at::kLong && beside(*ids) && (!mask || ((mask->scalar_type() == at::kBool || mask->scalar_type() == at::kByte) && beside(*mask)));
  });
  m.def("token_logprobs", [](const Tensor &x, const Tensor &ids, const std::optional<Tensor> &mask, double temperature) {
    const bool wanted = at::GradMode::is_enabled() && x.requires_grad();
    return unlocked([&] { return TokenLogprobs::apply(x, ids, mask, temperature, wanted); });
  });
  m.def("cross_entropy", [](const Tensor &x, const Tensor &ids, const std::optional<Tensor> &mask, int64_t reduction) {
    const bool wanted = at::GradMode::is_enabled() && x.requires_grad();
    return unlocked([&] { return CrossEntropy::apply(x, ids, mask, reduction, wanted); });
  });
  m.def("policy_loss", [](const Tensor &x, const Tensor &ids, const std::optional<Tensor> &mask, const std::optional<Tensor> &old_logps,
                          const Tensor &advantages, const std::optional<Tensor> &ref_logps, double clip_low, double clip_high, double kl_weight,
                          double temperature, int64_t reduction) {
    const bool wanted = at::GradMode::is_enabled() && x.requires_grad();
    const variable_list o = unlocked([&] {
      return PolicyLoss::apply(x, ids, mask, apart(old_logps), apart(advantages), apart(ref_logps), clip_low, clip_high, kl_weight, temperature,
                               reduction, wanted);
    });
    return py::make_tuple(wrap(o[0]), wrap(o[1]), wrap(o[2]));
  });
  m.def("preference_loss", [](const Tensor &x, const Tensor &ids, const std::optional<Tensor> &mask, const std::optional<Tensor> &ref_logps,
                              int64_t kind, double beta, double label_smoothing, bool average) {
    const bool wanted = at::GradMode::is_enabled() && x.requires_grad();
    const variable_list o = unlocked([&] {
      return PreferenceLoss::apply(x, ids, mask, apart(ref_logps), kind, beta, label_smoothing, average, wanted);
    });
    return py::make_tuple(wrap(o[0]), wrap(o[1]));
  });
  m.def("grad_norm", [](const Tensors &grads) { return unlocked([&] { return grad_norm(grads); }); });
  m.def("adamw_step", [](const Tensors &params, const Tensors &grads, const Tensors &exp_avgs, const Tensors &exp_avg_sqs, const Tensor &step,
                         const Tensors &scales, const Tensors &masters, const std::optional<Tensor> &lr_device, double lr, double beta1,
                         double beta2, double eps, double weight_decay, double max_grad_norm, bool skip_nonfinite,
                         const std::optional<Tensor> &norm, int64_t seed) {
    return wrap(unlocked([&] {
      return adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, scales, masters, given(lr_device), lr, beta1, beta2, eps, weight_decay,
                        max_grad_norm, skip_nonfinite, given(norm), seed);
    }));
  });
  m.def("forward_gn_gate", [](int64_t H, const std::optional<Tensor> &map, const Tensor &r, const Tensor &k, const Tensor &v, const Tensor &w,
                              const Tensor &u, const std::optional<Tensor> &s0, const Tensor &gate, const Tensor &scale,
                              const Tensor &offset, double eps, bool want_state) {
    return wrap(unlocked([&] {
      return forward_gn_gate(H, given(map), r, k, v, w, u, given(s0), gate, scale, offset, eps, want_state);
    }));
  });
}
