// The host side of group norm + activation, linear + activation + residual and the 8-bit activation checkpoints: argument
// checks, outputs, work buffers and the autograd nodes around the C ABI of libsg2im_hip.so.  These calls are short - a few
// microseconds on the GPU for a graph's objects - and from Python their checks, allocations and the backward pass' way
// through the interpreter took 24 us (forward) and 150 - 190 us (forward and backward); from here 6 and 65 - 75, of which
// torch.autograd.grad itself is some 35.
//
// Work buffers come from torch's allocator per call (inside a capture: from the graph's own pool), so neither two streams
// nor two captured graphs share one.  The library's entry points are bound by address (bind), so that this module uses
// whichever build of it the process has loaded.
#include <torch/extension.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <atomic>
#include <cmath>
#include <string>
#include <tuple>
#include <unordered_map>
#include "sg2im_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> MaybeTensor;

// ---- the library ------------------------------------------------------------------------------------------------------
struct Api {
  decltype(&sg2im_init) init;
  decltype(&sg2im_groupnorm_workspace) groupnorm_workspace;
  decltype(&sg2im_groupnorm_act_forward) groupnorm_act_forward;
  decltype(&sg2im_groupnorm_act_backward) groupnorm_act_backward;
  decltype(&sg2im_pack8) pack8;
  decltype(&sg2im_unpack8) unpack8;
  decltype(&sg2im_linear_workspace) linear_workspace;
  decltype(&sg2im_linear_backward_act_first) linear_backward_act_first;
  decltype(&sg2im_linear_forward) linear_forward;
  decltype(&sg2im_linear_backward_act) linear_backward_act;
  decltype(&sg2im_linear_backward_data) linear_backward_data;
  decltype(&sg2im_linear_backward_weight) linear_backward_weight;
} api;

void bind(const std::unordered_map<std::string, uintptr_t>& at) {
  #define SG2IM_BIND(f) api.f = reinterpret_cast<decltype(api.f)>(at.at("sg2im_" #f))
  SG2IM_BIND(init); SG2IM_BIND(groupnorm_workspace); SG2IM_BIND(groupnorm_act_forward); SG2IM_BIND(groupnorm_act_backward);
  SG2IM_BIND(pack8); SG2IM_BIND(unpack8); SG2IM_BIND(linear_workspace); SG2IM_BIND(linear_backward_act_first); SG2IM_BIND(linear_forward);
  SG2IM_BIND(linear_backward_act); SG2IM_BIND(linear_backward_data); SG2IM_BIND(linear_backward_weight);
  #undef SG2IM_BIND
}

void done(int status, const char* what) {
  TORCH_CHECK(status == SG2IM_OK, what, " failed: ", status == SG2IM_ERR_ARG ? "invalid argument" : "HIP runtime error");
}

const c10::impl::VirtualGuardImpl& gpu() {
  static const c10::impl::VirtualGuardImpl impl(c10::DeviceType::CUDA);
  return impl;
}

// ---- launches ---------------------------------------------------------------------------------------------------------
// The framework follows its launches: it counts the eager ones, times them by kind and prints them (_lib.call, ops._timed).  Those of
// this module are counted here - the backward passes' too, which no Python sees - and, while it is watched, announced to the
// observer before and after: observer(name, kind, amount, None) -> token, observer(name, kind, amount, token).
std::atomic<long long> eager_launches{0};
std::atomic<bool> watched{false};
PyObject* observer = nullptr;            // (held until the process ends)

void notify(const char* name, const char* kind, double amount, py::object& token) {
  token = py::reinterpret_borrow<py::object>(observer)(name, kind, amount, token);
}

// t's current stream, for a launch (the library's one-time set-up comes first)
hipStream_t stream_of(const Tensor& t) {
  static const int ready = api.init();
  done(ready, "sg2im_init");
  const c10::hip::HIPStream now = c10::hip::getCurrentHIPStream(t.device().index());
  hipStreamCaptureStatus status;               // (the default stream takes part in no capture, and is not to be asked during one)
  if (now == c10::hip::getDefaultHIPStream(t.device().index()) || hipStreamIsCapturing(now.stream(), &status) != hipSuccess ||
      status == hipStreamCaptureStatusNone) ++eager_launches;
  return now.stream();
}

// kind, amount: as ops._timed's (flops of the products, bytes of the others)
template <typename F> void launch(const char* name, const char* kind, double amount, const Tensor& on, F call) {
  const hipStream_t stream = stream_of(on);
  if (!watched) { done(call(stream), name); return; }
  py::gil_scoped_acquire gil;
  py::object token = py::none();
  notify(name, kind, amount, token);
  const int result = call(stream);
  notify(name, kind, amount, token);
  done(result, name);
}

// ---- checks -----------------------------------------------------------------------------------------------------------
bool is_bf16(const Tensor& t) { return t.scalar_type() == at::kBFloat16; }
int code(const Tensor& t) { return is_bf16(t) ? 1 : 0; }
at::ScalarType type_of(int c) { return c ? at::kBFloat16 : at::kFloat; }

void on_device(const Tensor& t, const char* what) {
  TORCH_CHECK_TYPE(t.is_cuda() && (t.scalar_type() == at::kFloat || is_bf16(t)), what,
                   ": expected a float32 / bfloat16 tensor on the GPU, got ", t.scalar_type(), " on ", t.device());
  TORCH_CHECK_VALUE(t.layout() == at::kStrided, what, ": expected a dense tensor");
  TORCH_CHECK_VALUE(!t.is_neg(), what, ": a view whose negation is pending (resolve_neg() makes it a tensor)");
  TORCH_CHECK_VALUE(t.device() == gpu().getDevice(), what, " lies on ", t.device(), " but the current device is ", gpu().getDevice());
}
// (a view whose negation is pending holds the numbers before it)
Tensor settled(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor given(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }

// These calls read and write memory below torch's dispatcher, so what follows operators there does not see them: a forward
// gradient would come back as none, that is as a derivative of zero, and a recorded program would hold the empty outputs and
// nothing that fills them.  Both are refused, before anything else is looked at.
void eager_only(const char* what, std::initializer_list<const Tensor*> tensors) {
  TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() &&
                              !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value(),
                              what, ": called while torch.jit.trace or make_fx records, which would not see it");
  for (const Tensor* t : tensors)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(),
                                what, ": no forward-mode derivative (an argument carries a forward gradient)");
}
const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* out_ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// the type of two parameter vectors of n values (either may be missing)
int params(const Tensor& weight, const Tensor& bias, int64_t n, const char* what) {
  int c = 0;
  for (const Tensor* t : {&weight, &bias}) {
    if (!t->defined()) continue;
    on_device(*t, what);
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == n && t->is_contiguous(), what, ": expected a dense vector of ", n, " values, got ", t->sizes());
    c = code(*t);
  }
  TORCH_CHECK_TYPE(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(), what, ": ",
                   weight.defined() ? weight.scalar_type() : at::kFloat, " and ", bias.defined() ? bias.scalar_type() : at::kFloat);
  return c;
}

Tensor work(const Tensor& like, size_t bytes) {
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte).memory_format(c10::nullopt));
}

// rows of t (..., C) as a matrix; a copy where they are not dense in memory
constexpr int64_t LD_MAX = 1 << 22;      // (the products' limit)
struct Rows { Tensor m; int64_t rows, cols, ld; };
Rows rows_of(const Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(t.dim() >= 1 && t.size(-1) >= 1, what, ": expected (..., channels), got ", t.sizes());
  Rows r;
  r.cols = t.size(-1);
  r.rows = t.numel() / r.cols;
  r.m = t.dim() == 2 ? t : t.is_contiguous() ? t.view({r.rows, r.cols}) : t.reshape({r.rows, r.cols});
  if ((r.cols > 1 && r.m.stride(1) != 1) || (r.rows > 1 && (r.m.stride(0) < r.cols || r.m.stride(0) > LD_MAX))) r.m = r.m.contiguous();
  r.ld = r.rows > 1 ? r.m.stride(0) : r.cols;
  return r;
}

int int_of(int64_t v, const char* what) {
  TORCH_CHECK_VALUE(v >= 0 && v <= 0x7fffffffLL, what, ": a size of ", v);
  return (int)v;
}

// ---- the 8-bit form ---------------------------------------------------------------------------------------------------
struct Packed { Tensor codes, exps; };
Packed packed_like(const Tensor& x) {
  auto shape = x.sizes().vec();
  Packed p;
  p.codes = at::empty(shape, x.options().dtype(at::kChar).memory_format(c10::nullopt));
  shape.back() = (shape.back() + 31) / 32;
  p.exps = at::empty(shape, x.options().dtype(at::kByte).memory_format(c10::nullopt));
  return p;
}
void check_packed(const Tensor& codes, const Tensor& exps, const char* what) {
  bool ok = codes.is_cuda() && exps.is_cuda() && codes.scalar_type() == at::kChar && exps.scalar_type() == at::kByte && codes.is_contiguous() &&
            exps.is_contiguous() && codes.dim() >= 1 && codes.size(-1) >= 1 && exps.dim() == codes.dim();
  for (int64_t d = 0; ok && d < codes.dim(); ++d) ok = exps.size(d) == (d + 1 < codes.dim() ? codes.size(d) : (codes.size(d) + 31) / 32);
  TORCH_CHECK_VALUE(ok, what, ": not an 8-bit form made by pack8");
  TORCH_CHECK_VALUE(codes.device() == gpu().getDevice() && exps.device() == codes.device(), what, ": the 8-bit form does not lie on the current device");
}
signed char* codes_ptr(const Tensor& t) { return t.defined() ? reinterpret_cast<signed char*>(t.data_ptr()) : nullptr; }
unsigned char* exps_ptr(const Tensor& t) { return t.defined() ? reinterpret_cast<unsigned char*>(t.data_ptr()) : nullptr; }

Packed pack(const Tensor& x) {
  on_device(x, "pack8");
  const Rows r = rows_of(x, "pack8");
  Packed p = packed_like(x);
  launch("sg2im_pack8", "hbm_pack8", x.numel() * (x.element_size() + 33.0 / 32), x, [&](hipStream_t stream) {
    return api.pack8(ptr(r.m), code(x), r.rows, int_of(r.cols, "pack8"), r.ld, codes_ptr(p.codes), exps_ptr(p.exps), stream);
  });
  return p;
}
std::tuple<Tensor, Tensor> pack8(const Tensor& x) {
  eager_only("pack8", {&x});
  const Packed p = pack(settled(x));
  return {p.codes, p.exps};
}

Tensor unpack8(const Tensor& codes, const Tensor& exps, int type) {
  eager_only("unpack8", {});
  check_packed(codes, exps, "unpack8");
  TORCH_CHECK_TYPE(type == 0 || type == 1, "unpack8: float32 or bfloat16");
  Tensor out = at::empty(codes.sizes(), codes.options().dtype(type_of(type)).memory_format(c10::nullopt));
  const int64_t C = codes.size(-1);
  launch("sg2im_unpack8", "hbm_unpack8", codes.numel() * (out.element_size() + 33.0 / 32), codes, [&](hipStream_t stream) {
    return api.unpack8(codes_ptr(codes), exps_ptr(exps), codes.numel() / C, int_of(C, "unpack8"), out_ptr(out), type, C, stream);
  });
  return out;
}

// ---- group norm + activation ------------------------------------------------------------------------------------------
struct GnShape { int n, c, g; long long hw; };
GnShape gn_shape(const Tensor& x, int64_t groups) {
  TORCH_CHECK_VALUE(x.dim() >= 2 && x.size(-1) >= 1, "group norm: expected (batch, ..., channels), got ", x.sizes());
  GnShape s;
  const int64_t C = x.size(-1);
  TORCH_CHECK_VALUE(groups >= 1 && C % groups == 0, "group norm: ", C, " channels do not divide into ", groups, " groups");
  s.hw = 1;
  for (int64_t d = 1; d + 1 < x.dim(); ++d) s.hw *= x.size(d);
  TORCH_CHECK_VALUE(s.hw >= 1, "group norm: an image without pixels ", x.sizes());
  s.n = int_of(x.size(0), "group norm"); s.c = int_of(C, "group norm"); s.g = (int)groups;
  return s;
}

struct GnResult { Tensor y, stats; Packed packed; };
GnResult gn_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t groups, double slope, double eps, int out_type, bool pack) {
  on_device(x, "group norm input");
  const GnShape s = gn_shape(x, groups);
  TORCH_CHECK_VALUE(x.is_contiguous(), "group norm: the input must be dense");
  if (out_type < 0) out_type = code(x);
  TORCH_CHECK_TYPE(out_type == 1 || !is_bf16(x), "group norm: a float32 output of a bfloat16 input");
  TORCH_CHECK_VALUE(eps >= 0 && std::isfinite((float)slope), "group norm: eps = ", eps, ", slope = ", slope);
  const int pc = params(weight, bias, s.c, "group norm parameters");
  const size_t bytes = api.groupnorm_workspace(s.n, s.hw, s.c, s.g, code(x), 0);
  TORCH_CHECK_VALUE(bytes, "group norm: ", x.sizes(), " is too large");
  GnResult r;
  r.y = at::empty(x.sizes(), x.options().dtype(type_of(out_type)).memory_format(c10::nullopt));
  r.stats = at::empty({s.n, s.g, 2}, x.options().dtype(at::kDouble).memory_format(c10::nullopt));
  if (pack) r.packed = packed_like(x);
  const Tensor w = work(x, bytes);
  launch("sg2im_groupnorm_act_forward", "hbm_group_norm_fwd", x.numel() * (x.element_size() + r.y.element_size() + (pack ? 33.0 / 32 : 0.0)), x, [&](hipStream_t stream) {
    return api.groupnorm_act_forward(ptr(x), code(x), s.n, s.hw, s.c, s.g, ptr(weight), ptr(bias), pc, (float)slope, (float)eps, out_ptr(r.y), out_type,
         reinterpret_cast<double*>(out_ptr(r.stats)), codes_ptr(r.packed.codes), exps_ptr(r.packed.exps), out_ptr(w), bytes,
         stream);
  });
  return r;
}

// x: the input, or undefined next to its 8-bit form; dweight / dbias: where those gradients go, or undefined
Tensor gn_backward(const Tensor& dy, const Tensor& x, const Packed& packed, int x_type, const Tensor& weight, const Tensor& bias, int64_t groups,
                   double slope, const Tensor& stats, bool need_dx, const Tensor& dweight, const Tensor& dbias, bool accumulate) {
  on_device(dy, "group norm gradient");
  if (x.defined()) on_device(x, "group norm input"); else check_packed(packed.codes, packed.exps, "group norm backward");
  const Tensor& shaped = x.defined() ? x : packed.codes;
  TORCH_CHECK_VALUE(dy.sizes() == shaped.sizes() && dy.is_contiguous() && shaped.is_contiguous(), "group norm backward: dense tensors of one shape, got ",
                    dy.sizes(), " and ", shaped.sizes());
  TORCH_CHECK_TYPE(x_type == 0 || is_bf16(dy), "group norm backward: a float32 gradient of a bfloat16 input");
  const GnShape s = gn_shape(dy, groups);
  const int pc = params(weight, bias, s.c, "group norm parameters"), gc = params(dweight, dbias, s.c, "group norm gradients");
  TORCH_CHECK_VALUE(stats.is_cuda() && stats.scalar_type() == at::kDouble && stats.is_contiguous() && stats.device() == dy.device() &&
                    stats.numel() == (int64_t)s.n * s.g * 2,
                    "group norm backward: not the statistics of this input");
  const size_t bytes = api.groupnorm_workspace(s.n, s.hw, s.c, s.g, x_type, 1);
  Tensor dx = need_dx ? at::empty(dy.sizes(), dy.options().dtype(type_of(x_type)).memory_format(c10::nullopt)) : Tensor();
  const Tensor w = work(dy, bytes);
  launch("sg2im_groupnorm_act_backward", "hbm_group_norm_bwd", dy.numel() * (dy.element_size() + (x.defined() ? x.element_size() : 33.0 / 32) + (need_dx ? dx.element_size() : 0.0)), dy, [&](hipStream_t stream) {
    return api.groupnorm_act_backward(ptr(dy), code(dy), ptr(x), x_type, codes_ptr(packed.codes), exps_ptr(packed.exps), s.n, s.hw, s.c, s.g, ptr(weight),
         ptr(bias), pc, (float)slope, reinterpret_cast<const double*>(ptr(stats)), out_ptr(dx), out_ptr(dweight),
         out_ptr(dbias), gc, accumulate, out_ptr(w), bytes, stream);
  });
  return dx;
}

// a parameter's gradient: its registered sink, or a new tensor
struct Target {
  Tensor buf; bool own;
  Target(bool need, const Tensor& like, const Tensor& sink) : own(false) {
    if (!need || !like.defined()) return;
    if (sink.defined()) buf = sink;
    else { buf = at::empty(like.sizes(), like.options().memory_format(c10::nullopt)); own = true; }
  }
  Tensor grad() const { return own ? buf : Tensor(); }
};

void once(const char* what, const Tensor& grad) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "this operator has no second derivative (create_graph=True reached its backward pass)");
  eager_only(what, {&grad});
}

// the registered gradient buffers of a layer's two parameters (undefined: none); autograd does not see them
struct Sinks {
  Tensor w, b;
  void keep(AutogradContext* ctx) const {
    if (w.defined()) ctx->saved_data["sink_w"] = w;
    if (b.defined()) ctx->saved_data["sink_b"] = b;
  }
  static Tensor kept(AutogradContext* ctx, const char* name) {
    const auto at = ctx->saved_data.find(name);
    return at == ctx->saved_data.end() ? Tensor() : at->second.toTensor();
  }
};
MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

struct GroupNormAct : torch::autograd::Function<GroupNormAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight_, const MaybeTensor& bias_, int64_t groups, double slope,
                        double eps, bool checkpoint8, int64_t out_type, const Sinks* sinks) {
    const Tensor weight = given(weight_), bias = given(bias_);
    const GnResult r = gn_forward(x, weight, bias, groups, slope, eps, (int)out_type, checkpoint8);
    ctx->save_for_backward({checkpoint8 ? Tensor() : x, r.packed.codes, r.packed.exps, weight, bias, r.stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["slope"] = slope;
    ctx->saved_data["type"] = (int64_t)code(x);
    sinks->keep(ctx);
    return r.y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("group norm backward", grads[0]);
    const variable_list s = ctx->get_saved_variables();
    // (edges are numbered over the tensors that are there)
    const bool nw = s[3].defined() && ctx->needs_input_grad(1), nb = s[4].defined() && ctx->needs_input_grad(s[3].defined() ? 2 : 1);
    Tensor sw = Sinks::kept(ctx, "sink_w"), sb = Sinks::kept(ctx, "sink_b");
    // one launch adds to both or writes both: a sink next to a parameter without one is added to afterwards
    const bool all = (!nw || sw.defined()) && (!nb || sb.defined());
    const Target tw(nw, s[3], all ? sw : Tensor()), tb(nb, s[4], all ? sb : Tensor());
    const Tensor dx = gn_backward(settled(grads[0]).contiguous(), s[0], Packed{s[1], s[2]}, (int)ctx->saved_data["type"].toInt(), s[3], s[4],
                                  ctx->saved_data["groups"].toInt(), ctx->saved_data["slope"].toDouble(), s[5], ctx->needs_input_grad(0),
                                  tw.buf, tb.buf, all);
    Tensor dw = tw.grad(), db = tb.grad();
    if (dw.defined() && sw.defined()) { sw.add_(dw); dw = Tensor(); }
    if (db.defined() && sb.defined()) { sb.add_(db); db = Tensor(); }
    return {dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

bool wants(const Tensor& t) { return t.defined() && t.requires_grad(); }

// A leaf's gradient is handed over on the stream on which its accumulation node was made, and that node lives as long as any
// graph of the leaf does.  Made on the default stream, which cannot take part in a capture, it would end the process in the
// captured backward pass: such a call is refused while it is recorded.  (With a sink nothing is handed over.)
void check_capture(std::initializer_list<std::pair<const Tensor*, const Tensor*>> leaves) {
  const c10::hip::HIPStream now = c10::hip::getCurrentHIPStream(), usual = c10::hip::getDefaultHIPStream();
  hipStreamCaptureStatus status;
  if (now == usual || hipStreamIsCapturing(now.stream(), &status) != hipSuccess || status == hipStreamCaptureStatusNone) return;
  for (const auto& [t, sink] : leaves) {
    if (!wants(*t) || !t->is_leaf() || (sink && sink->defined())) continue;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
    const auto stream = node ? node->stream() : c10::nullopt;
    TORCH_CHECK(!stream.has_value() || stream->id() != usual.id(),
                "captured into a graph while a gradient graph of the same leaf, made on the default stream, is alive: release it before the "
                "capture, or record with a detached copy of the leaf");
  }
}

Tensor group_norm_act(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, int64_t groups, double slope, double eps, bool checkpoint8,
                      int64_t out_type, const MaybeTensor& sink_w, const MaybeTensor& sink_b) {
  const Tensor w = given(weight), b = given(bias);
  eager_only("group norm", {&x, &w, &b});
  if (!(at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b))))
    return gn_forward(settled(x).contiguous(), w, b, groups, slope, eps, (int)out_type, false).y;
  const Sinks sinks{given(sink_w), given(sink_b)};
  check_capture({{&x, nullptr}, {&w, &sinks.w}, {&b, &sinks.b}});
  return GroupNormAct::apply(settled(x).contiguous(), maybe(w), maybe(b), groups, slope, eps, checkpoint8, out_type, &sinks);
}

// ---- linear + activation + residual -----------------------------------------------------------------------------------
void check_weight(const Tensor& w, at::ScalarType type) {
  on_device(w, "linear weight");
  TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) >= 1 && w.size(1) >= 1 && w.is_contiguous() && w.scalar_type() == type,
                    "linear: the weight must be a dense matrix of the input's type ", type, ", got ", w.scalar_type(), " ", w.sizes());
}

std::tuple<Tensor, Tensor> lin_forward(const Tensor& x, const Tensor& weight, const Tensor& bias, const Tensor& residual, double slope, int out_type,
                                       bool want_signs) {
  on_device(x, "linear input");
  check_weight(weight, x.scalar_type());
  const int N = int_of(weight.size(0), "linear"), K = int_of(weight.size(1), "linear");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == K, "linear: input ", x.sizes(), " and weight ", weight.sizes());
  if (out_type < 0) out_type = code(x);
  TORCH_CHECK_TYPE(out_type == 0 || is_bf16(x), "linear: a bfloat16 output of float32 operands");
  TORCH_CHECK_VALUE(std::isfinite((float)slope), "linear: slope = ", slope);
  const int bc = params(Tensor(), bias, N, "linear bias");
  const Rows r = rows_of(x, "linear input");
  auto shape = x.sizes().vec();
  shape.back() = N;
  Rows res;
  res.ld = N;
  if (residual.defined()) {
    on_device(residual, "linear residual");
    TORCH_CHECK_VALUE(residual.sizes() == at::IntArrayRef(shape) && residual.scalar_type() == type_of(out_type), "linear: the residual must be ",
                      type_of(out_type), " ", shape, ", got ", residual.scalar_type(), " ", residual.sizes());
    res = rows_of(residual, "linear residual");
  }
  Tensor y = at::empty(shape, x.options().dtype(type_of(out_type)).memory_format(c10::nullopt)), signs;
  if (want_signs) signs = at::empty({r.rows, (N + 31) / 32}, x.options().dtype(at::kInt).memory_format(c10::nullopt));
  const size_t bytes = api.linear_workspace(r.rows, K, N, code(x), 0);
  const Tensor w = work(x, bytes);
  launch("sg2im_linear_forward", "igemm_fwd", 2.0 * r.rows * K * N, x, [&](hipStream_t stream) {
    return api.linear_forward(ptr(r.m), code(x), r.ld, ptr(weight), ptr(bias), bc, ptr(res.m), res.ld, (float)slope, out_ptr(y), out_type, N,
         reinterpret_cast<unsigned*>(out_ptr(signs)), r.rows, K, N, out_ptr(w), bytes, stream);
  });
  return {y, signs};
}

void check_signs(const Tensor& signs, const Rows& dy) {
  TORCH_CHECK_VALUE(!signs.defined() || (signs.is_cuda() && signs.scalar_type() == at::kInt && signs.is_contiguous() && signs.dim() == 2 &&
                                         signs.device() == dy.m.device() && signs.size(0) == dy.rows && signs.size(1) == (dy.cols + 31) / 32), "linear backward: not the signs of this output");
}
const unsigned* signs_ptr(const Tensor& t) { return reinterpret_cast<const unsigned*>(ptr(t)); }

// dz in `dz_type` (-1: not written) and the bias gradient into dbias (undefined: none)
Tensor lin_backward_act(const Rows& dy, const Tensor& signs, double slope, int dz_type, const Tensor& dbias, bool accumulate) {
  const int N = int_of(dy.cols, "linear gradient");
  check_signs(signs, dy);
  TORCH_CHECK_TYPE(dz_type != 0 || !is_bf16(dy.m), "linear backward: a float32 dz of a bfloat16 gradient");
  const int bc = params(Tensor(), dbias, N, "linear bias gradient");
  Tensor dz;
  if (dz_type >= 0) dz = at::empty({dy.rows, dy.cols}, dy.m.options().dtype(type_of(dz_type)).memory_format(c10::nullopt));
  const size_t bytes = api.linear_workspace(dy.rows, 1, N, 0, 3);
  const Tensor w = work(dy.m, bytes);
  launch("sg2im_linear_backward_act", "hbm_linear_act_bwd", (double)dy.rows * N * (dy.m.element_size() + (dz.defined() ? dz.element_size() : 0.0)), dy.m, [&](hipStream_t stream) {
    return api.linear_backward_act(ptr(dy.m), code(dy.m), dy.ld, reinterpret_cast<const unsigned*>(ptr(signs)), (float)slope, out_ptr(dz),
         dz_type < 0 ? code(dy.m) : dz_type, out_ptr(dbias), bc, accumulate, dy.rows, N, out_ptr(w), bytes, stream);
  });
  return dz;
}

Tensor lin_backward_data(const Rows& dz, const Tensor& signs, double slope, const Tensor& weight, at::IntArrayRef shape) {
  check_signs(signs, dz);
  check_weight(weight, dz.m.scalar_type());
  TORCH_CHECK_VALUE(weight.size(0) == dz.cols, "linear backward: gradient ", dz.m.sizes(), " and weight ", weight.sizes());
  const int N = (int)weight.size(0), K = int_of(weight.size(1), "linear");
  Tensor dx = at::empty(shape, dz.m.options().memory_format(c10::nullopt));
  const size_t bytes = api.linear_workspace(dz.rows, K, N, code(dz.m), 1);
  const Tensor w = work(dz.m, bytes);
  launch("sg2im_linear_backward_data", "igemm_dgrad", 2.0 * dz.rows * K * N, dz.m, [&](hipStream_t stream) {
    return api.linear_backward_data(ptr(dz.m), code(dz.m), dz.ld, signs_ptr(signs), (float)slope, ptr(weight), out_ptr(dx), K, dz.rows, K, N, out_ptr(w), bytes, stream);
  });
  return dx;
}

void lin_backward_weight(const Rows& dz, const Tensor& signs, double slope, const Tensor& x, const Packed& packed, const Tensor& dweight,
                         bool accumulate, const Tensor& dbias, bool bias_accumulate) {
  check_signs(signs, dz);
  const int bc = params(Tensor(), dbias, dz.cols, "linear bias gradient");
  on_device(dweight, "linear weight gradient");
  Rows r;
  if (x.defined()) {
    on_device(x, "linear input");
    TORCH_CHECK_TYPE(x.scalar_type() == dz.m.scalar_type(), "linear backward: gradient ", dz.m.scalar_type(), ", input ", x.scalar_type());
    r = rows_of(x, "linear input");
  } else {
    check_packed(packed.codes, packed.exps, "linear backward");
    r.cols = packed.codes.size(-1);
    r.rows = packed.codes.numel() / r.cols;
    r.ld = r.cols;
  }
  const int N = int_of(dz.cols, "linear gradient"), K = int_of(r.cols, "linear input");
  TORCH_CHECK_VALUE(r.rows == dz.rows && dweight.dim() == 2 && dweight.size(0) == N && dweight.size(1) == K && dweight.is_contiguous() &&
                    (dweight.scalar_type() == at::kFloat || is_bf16(dz.m)), "linear backward: gradient of ", dz.rows, " x ", dz.cols, ", input of ",
                    r.rows, " x ", r.cols, ", weight gradient ", dweight.scalar_type(), " ", dweight.sizes());
  const size_t bytes = api.linear_workspace(dz.rows, K, N, code(dz.m), 2);
  const Tensor w = work(dz.m, bytes);
  launch("sg2im_linear_backward_weight", "igemm_wgrad", 2.0 * dz.rows * K * N, dz.m, [&](hipStream_t stream) {
    return api.linear_backward_weight(ptr(dz.m), code(dz.m), dz.ld, signs_ptr(signs), (float)slope, ptr(r.m), r.ld, codes_ptr(packed.codes),
         exps_ptr(packed.exps), out_ptr(dweight), code(dweight), accumulate, out_ptr(dbias), bc, bias_accumulate, dz.rows, K, N, out_ptr(w), bytes, stream);
  });
}

struct LinearResidual : torch::autograd::Function<LinearResidual> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const MaybeTensor& bias_, const MaybeTensor& residual, double slope,
                        bool checkpoint8, int64_t out_type, const Sinks* sinks) {
    const Tensor bias = given(bias_);
    Tensor w = weight.contiguous();
    if (is_bf16(x) && w.scalar_type() == at::kFloat) w = w.to(at::kBFloat16);
    const bool for_w = weight.requires_grad(), gates = slope != 1.0 && (for_w || wants(x) || wants(bias));
    auto [y, signs] = lin_forward(x, w, bias, given(residual), slope, (int)out_type, gates);
    Packed p;
    if (checkpoint8 && for_w) p = pack(x);
    ctx->save_for_backward({for_w && !checkpoint8 ? x : Tensor(), p.codes, p.exps, weight, w.is_same(weight) ? Tensor() : w, bias, signs});
    ctx->saved_data["slope"] = slope;
    ctx->saved_data["residual"] = residual.has_value();
    ctx->saved_data["type"] = (int64_t)code(x);
    ctx->saved_data["shape"] = x.sizes().vec();
    sinks->keep(ctx);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("linear backward", grads[0]);
    const variable_list s = ctx->get_saved_variables();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1), nb = s[5].defined() && ctx->needs_input_grad(2);
    const bool nr = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(s[5].defined() ? 3 : 2);
    const int type = (int)ctx->saved_data["type"].toInt();
    const Tensor& signs = s[6];
    Tensor dx, dw, db;
    if (nx || nw || nb) {
      const Tensor given_dy = settled(grads[0]);
      on_device(given_dy, "linear gradient");
      const Rows dy = rows_of(given_dy, "linear gradient");
      const double slope = ctx->saved_data["slope"].toDouble();
      const Target tb(nb, s[5], Sinks::kept(ctx, "sink_b"));
      // dz = dy * leaky' and the bias gradient: a pass of their own, or done by the products as they read dy
      const bool same = code(dy.m) == type, products = nx || nw;
      const bool first = products && same && api.linear_backward_act_first(dy.rows, (int)s[3].size(1), (int)s[3].size(0), type, signs.defined(),
                                                                           nb, nx, nw);
      const bool own = products && (!same || (first && signs.defined()));
      Rows dz = dy;
      Tensor gate = signs;
      bool summed = false;
      if (own || (nb && (!nw || first))) {
        const Tensor z = lin_backward_act(dy, signs, slope, own ? type : -1, tb.buf, !tb.own);
        summed = true;
        if (own) { dz.m = z; dz.ld = dz.cols; gate = Tensor(); }
      }
      if (nx) dx = lin_backward_data(dz, gate, slope, s[4].defined() ? s[4] : s[3], ctx->saved_data["shape"].toIntVector());
      if (nw) {
        const Target tw(true, s[3], Sinks::kept(ctx, "sink_w"));
        lin_backward_weight(dz, gate, slope, s[0], Packed{s[1], s[2]}, tw.buf, !tw.own, summed ? Tensor() : tb.buf, !tb.own);
        dw = tw.grad();
      }
      db = tb.grad();
    }
    return {dx, dw, db, nr ? grads[0] : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor linear_residual(const Tensor& x_, const Tensor& weight_, const MaybeTensor& bias, const MaybeTensor& residual, double slope, bool checkpoint8,
                       int64_t out_type, const MaybeTensor& sink_w, const MaybeTensor& sink_b) {
  const Tensor b = given(bias);
  Tensor x = x_, weight = weight_, r = given(residual);
  eager_only("linear", {&x, &weight, &b, &r});
  for (Tensor* t : {&x, &weight, &r}) if (t->defined()) *t = settled(*t);
  if (!(at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(b) || wants(r)))) {
    Tensor w = weight.contiguous();
    if (is_bf16(x) && w.scalar_type() == at::kFloat) w = w.to(at::kBFloat16);
    return std::get<0>(lin_forward(x, w, b, r, slope, (int)out_type, false));
  }
  const Sinks sinks{given(sink_w), given(sink_b)};
  check_capture({{&x, nullptr}, {&weight, &sinks.w}, {&b, &sinks.b}, {&r, nullptr}});
  return LinearResidual::apply(x, weight, maybe(b), maybe(r), slope, checkpoint8, out_type, &sinks);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("observe", [](py::object f) { observer = f.release().ptr(); });
  m.def("watch", [](bool on) { watched = on && observer; });
  m.def("eager_launches", [] { return eager_launches.load(); });
  m.def("pack8", &pack8);
  m.def("unpack8", &unpack8);
  m.def("group_norm_act", &group_norm_act);
  m.def("linear_residual", &linear_residual);
  // the passes on their own (missing tensors: None)
  m.def("group_norm_act_forward", [](const Tensor& x, const MaybeTensor& w, const MaybeTensor& b, int64_t groups, double slope, double eps,
                                     int64_t out_type, bool pack) {
    const Tensor wt = given(w), bt = given(b);
    eager_only("group norm", {&x, &wt, &bt});
    const GnResult r = gn_forward(x, wt, bt, groups, slope, eps, (int)out_type, pack);
    return std::make_tuple(r.y, r.stats, r.packed.codes, r.packed.exps);
  });
  m.def("group_norm_act_backward", [](const Tensor& dy, const MaybeTensor& x, const MaybeTensor& codes, const MaybeTensor& exps, int64_t x_type,
                                      const MaybeTensor& w, const MaybeTensor& b, int64_t groups, double slope, const Tensor& stats, bool need_dx,
                                      const MaybeTensor& dw, const MaybeTensor& db, bool accumulate) {
    const Tensor xt = given(x), wt = given(w), bt = given(b), dwt = given(dw), dbt = given(db);
    eager_only("group norm backward", {&dy, &xt, &wt, &bt, &stats, &dwt, &dbt});
    return gn_backward(dy, xt, Packed{given(codes), given(exps)}, (int)x_type, wt, bt, groups, slope, stats, need_dx, dwt, dbt, accumulate);
  });
  m.def("linear_forward", [](const Tensor& x, const Tensor& w, const MaybeTensor& b, const MaybeTensor& r, double slope, int64_t out_type, bool signs) {
    const Tensor bt = given(b), rt = given(r);
    eager_only("linear", {&x, &w, &bt, &rt});
    return lin_forward(x, w, bt, rt, slope, (int)out_type, signs);
  });
  m.def("linear_backward_act", [](const Tensor& dy, const MaybeTensor& signs, double slope, int64_t dz_type, const MaybeTensor& db, bool accumulate) {
    const Tensor dbt = given(db);
    eager_only("linear backward", {&dy, &dbt});
    on_device(dy, "linear gradient");
    return lin_backward_act(rows_of(dy, "linear gradient"), given(signs), slope, (int)dz_type, dbt, accumulate);
  });
  m.def("linear_backward_data", [](const Tensor& dz, const Tensor& w, const MaybeTensor& signs, double slope) {
    eager_only("linear backward", {&dz, &w});
    on_device(dz, "linear gradient");
    const Rows r = rows_of(dz, "linear gradient");
    return lin_backward_data(r, given(signs), slope, w, {r.rows, w.size(-1)});
  });
  m.def("linear_backward_weight", [](const Tensor& dz, const MaybeTensor& x, const MaybeTensor& codes, const MaybeTensor& exps, const Tensor& dw,
                                     bool accumulate, const MaybeTensor& db, bool bias_accumulate, const MaybeTensor& signs, double slope) {
    const Tensor xt = given(x), dbt = given(db);
    eager_only("linear backward", {&dz, &xt, &dw, &dbt});
    on_device(dz, "linear gradient");
    lin_backward_weight(rows_of(dz, "linear gradient"), given(signs), slope, xt, Packed{given(codes), given(exps)}, dw, accumulate, dbt, bias_accumulate);
  });
}
