// Autograd nodes and argument checks of layer_norm, dropout and gated_ffn: what their Python entry points call.
//
// The one file that is compiled against PyTorch's headers (host code only; the kernels stay behind the C ABI of block_calls.h).
// A training call of these operators on small tensors is bound by the host, and a node written in Python costs it about
// 40 us more: its backward function has to take the interpreter's lock in the engine's thread, and allocations, views and the
// call cost several times what they do here.  1120 x 650 fp32 layer norm, forward and backward: 114 us with Python nodes, 72 with these.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include <atomic>
#include <optional>
#include <sstream>

#include "block_calls.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

std::atomic<long long> g_launches{0};      // kernels launched by the calls below

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? 0 : (t == at::kBFloat16 ? 1 : (t == at::kHalf ? 2 : -1));
}
void check(int rc, const char* what) {
  if (rc == 0) return;
  std::ostringstream s;
  s << what << " failed with code " << rc;
  if (rc > 0) s << " (" << choco_cuda_error_string(rc) << ")";
  throw std::runtime_error(s.str());
}
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
std::string describe(const Tensor& t) {
  std::ostringstream s;
  if (!t.defined()) return "None";
  s << t.sizes() << " " << t.scalar_type() << " " << t.device();
  return s.str();
}
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
// a tangent of forward-mode differentiation: the kernels would drop it without a word
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
void no_tangent(const char* what, std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(*t), what, ": no forward-mode derivative (an input or a gradient carries a tangent)");
}
void no_second_derivative(const char* what) {
  if (at::GradMode::is_enabled())
    throw std::runtime_error(std::string(what) + ": the backward kernels have no derivative (create_graph=True)");
}

// t as [rows, last] with a contiguous last dimension: a view where the strides allow it
Tensor rows_of(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return r.stride(1) == 1 && r.stride(0) >= r.size(1) ? r : r.contiguous();
}
// elements from row to row (a single row's stride says nothing)
long long pitch(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max<long long>(1, t.size(1)); }
// Saved tensors come back through hooks (offloading, recomputation), and a leaf's .data can be assigned to in between: the
// values are the same, strides and alignment need not be.  Size, type and device have to.
void check_saved(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type, const at::Device& device, const char* what) {
  if (t.defined() && t.sizes() == sizes && t.scalar_type() == type && t.device() == device) return;
  std::ostringstream s;
  s << what << ": a saved tensor came back as " << describe(t) << ", it was " << sizes << " " << type << " " << device;
  throw std::runtime_error(s.str());
}
// a workspace as the kernels need it: one run of bytes on a 256-byte boundary
Tensor workspace_of(const Tensor& t) {
  if (t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 256 == 0) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}
Tensor empty(at::IntArrayRef sizes, const Tensor& like) { return at::empty(sizes, like.options()); }
Tensor empty_floats(long long n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kFloat)); }

// ---- layer norm -----------------------------------------------------------------------------------------------------
bool layer_norm_ok(const Tensor& x, const Tensor& w, const Tensor& b) {
  if (!x.is_cuda() || dtype_code(x.scalar_type()) < 0 || x.dim() < 1 || x.size(-1) < 1 || x.size(-1) >= (1 << 24)) return false;
  for (const Tensor* p : {&w, &b})
    if (p->defined() && !(p->dim() == 1 && p->size(0) == x.size(-1) && p->device() == x.device() &&
                          (p->scalar_type() == x.scalar_type() || p->scalar_type() == at::kFloat)))
      return false;
  return !w.defined() || !b.defined() || w.scalar_type() == b.scalar_type();
}

Tensor layer_norm_run(const Tensor& x, const Tensor& x2, const Tensor& w, const Tensor& b, double eps, const Tensor& stats) {
  Tensor y = empty(x.sizes(), x);
  const Tensor& p = w.defined() ? w : b;
  LnForwardCall c = {};
  c.x = x2.data_ptr(); c.ldx = pitch(x2); c.w = ptr(w); c.b = ptr(b); c.y = y.data_ptr();
  c.stats = reinterpret_cast<float*>(ptr(stats));
  c.n = x2.size(0); c.d = x2.size(1); c.dt = dtype_code(x.scalar_type());
  c.w_dt = p.defined() ? dtype_code(p.scalar_type()) : c.dt;
  c.eps = eps;
  c.stream = stream_of(x);
  if (c.n > 0) {
    check(layer_norm_forward(&c), "layer_norm_forward");
    g_launches += c.launches;
  }
  return y;
}

// An absent tensor goes into Function::apply as an empty optional; needs_input_grad counts the ones that are there.
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }

struct LayerNormFn : torch::autograd::Function<LayerNormFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    ctx->saved_data["bias"] = b.defined();
    const Tensor x2 = rows_of(x), stats = empty_floats(2 * x2.size(0), x);
    ctx->save_for_backward({x2, w, stats});
    ctx->saved_data["type"] = static_cast<int64_t>((w.defined() ? w : (b.defined() ? b : x)).scalar_type());
    ctx->saved_data["rows"] = x2.size(0);
    return layer_norm_run(x, x2, w, b, eps, stats);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative("layer_norm");
    no_tangent("layer_norm", {&grads[0]});
    const variable_list saved = ctx->get_saved_variables();
    const Tensor dy2 = rows_of(grads[0]);
    const int64_t rows = ctx->saved_data["rows"].toInt(), width = dy2.size(1);
    const auto type = static_cast<at::ScalarType>(ctx->saved_data["type"].toInt());
    check_saved(saved[0], {rows, width}, dy2.scalar_type(), dy2.device(), "layer_norm");
    if (saved[1].defined()) check_saved(saved[1], {width}, type, dy2.device(), "layer_norm");
    check_saved(saved[2], {2 * rows}, at::kFloat, dy2.device(), "layer_norm");
    const c10::OptionalDeviceGuard guard(dy2.device());
    const Tensor x2 = rows_of(saved[0]), w = saved[1].defined() ? saved[1].contiguous() : saved[1], stats = saved[2].contiguous();
    Tensor dx, dw, db, partial;
    if (ctx->needs_input_grad(0)) dx = empty(grads[0].sizes(), x2);
    const size_t bias_index = w.defined() ? 2 : 1;
    if (w.defined() && ctx->needs_input_grad(1)) dw = at::empty({x2.size(1)}, x2.options().dtype(type));
    if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(bias_index)) db = at::empty({x2.size(1)}, x2.options().dtype(type));
    LnBackwardCall c = {};
    c.n = x2.size(0); c.d = x2.size(1);
    if (c.n == 0) {
      if (dw.defined()) dw.zero_();
      if (db.defined()) db.zero_();
      return {dx, dw, db, Tensor()};
    }
    if (dw.defined() || db.defined()) partial = empty_floats(layer_norm_partial_floats((int)c.d), x2);
    c.x = x2.data_ptr(); c.ldx = pitch(x2); c.dy = dy2.data_ptr(); c.lddy = pitch(dy2); c.w = ptr(w);
    c.stats = stats.data_ptr<float>();
    c.dx = ptr(dx); c.dw = ptr(dw); c.db = ptr(db);
    c.partial = reinterpret_cast<float*>(ptr(partial));
    c.dt = dtype_code(x2.scalar_type()); c.w_dt = dtype_code(type);
    c.stream = stream_of(x2);
    check(layer_norm_backward(&c), "layer_norm_backward");
    g_launches += c.launches;
    return {dx, dw, db, Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const Maybe& weight, const Maybe& bias, double eps) {
  Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  if (!layer_norm_ok(x, w, b))
    throw pybind11::value_error(
        "layer_norm: needs a CUDA tensor of fp32, bf16 or fp16 and, where given, weight and bias of its last dimension's length on "
        "its device, both of its type or both fp32: got " + describe(x) + ", " + describe(w) + ", " + describe(b));
  no_tangent("layer_norm", {&x, &w, &b});
  const c10::OptionalDeviceGuard guard(x.device());
  if (w.defined()) w = w.contiguous();
  if (b.defined()) b = b.contiguous();
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b))) return LayerNormFn::apply(x, maybe(w), maybe(b), eps);
  return layer_norm_run(x, rows_of(x), w, b, eps, Tensor());
}

// ---- dropout --------------------------------------------------------------------------------------------------------
Tensor dropout_run(const Tensor& in, const Tensor& residual, const Tensor& key, int64_t drop, int64_t site) {
  const Tensor x = in.contiguous(), r = residual.defined() ? residual.contiguous() : residual;
  Tensor y = empty(x.sizes(), x);
  DropoutCall c = {};
  c.x = x.data_ptr(); c.res = ptr(r); c.y = y.data_ptr(); c.n = x.numel(); c.key = key.data_ptr();
  c.site = site; c.drop = drop; c.dt = dtype_code(x.scalar_type());
  c.stream = stream_of(x);
  if (c.n > 0) {
    check(dropout_apply(&c), "dropout_apply");
    g_launches += c.launches;
  }
  return y;
}

struct DropoutFn : torch::autograd::Function<DropoutFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& residual, const Tensor& key, int64_t drop, int64_t site) {
    ctx->save_for_backward({key});
    ctx->saved_data["drop"] = drop;
    ctx->saved_data["site"] = site;
    ctx->saved_data["residual"] = residual.has_value();
    return dropout_run(x, residual.value_or(Tensor()), key, drop, site);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor key = ctx->get_saved_variables()[0], &dy = grads[0];
    no_tangent("dropout", {&dy});
    static const int64_t one = 1;
    check_saved(key, key.numel() == 1 ? key.sizes() : at::IntArrayRef(one), at::kLong, dy.device(), "dropout");
    const int64_t drop = ctx->saved_data["drop"].toInt(), site = ctx->saved_data["site"].toInt();
    const c10::OptionalDeviceGuard guard(dy.device());
    Tensor dx, dr;
    if (ctx->needs_input_grad(0))      // the gradient's gradient is the same function again
      dx = at::GradMode::is_enabled() ? DropoutFn::apply(dy, Maybe(), key, drop, site) : dropout_run(dy, Tensor(), key, drop, site);
    if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(1)) dr = dy;
    return {dx, dr, Tensor(), Tensor(), Tensor()};
  }
};

// drop: the probability in steps of 2^-16, 0 .. 65536
Tensor dropout(const Tensor& x, int64_t drop, const Tensor& key, int64_t site, const Maybe& res) {
  const Tensor residual = res.value_or(Tensor());
  if (!x.is_cuda() || dtype_code(x.scalar_type()) < 0)
    throw pybind11::value_error("dropout: needs a CUDA tensor of fp32, bf16 or fp16, got " + describe(x));
  if (!(key.scalar_type() == at::kLong && key.numel() == 1 && key.device() == x.device()))
    throw pybind11::value_error("dropout: the key is one 64-bit integer on the input's device (new_key), got " + describe(key));
  if (residual.defined() && !(residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type() && residual.device() == x.device()))
    throw pybind11::value_error("dropout: the residual has the input's shape, type and device, got " + describe(residual) + " for " + describe(x));
  no_tangent("dropout", {&x, &residual});
  const c10::OptionalDeviceGuard guard(x.device());
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(residual))) return DropoutFn::apply(x, maybe(residual), key, drop, site);
  return dropout_run(x, residual, key, drop, site);
}

// ---- gated feed-forward ---------------------------------------------------------------------------------------------
long long pad(long long n, long long to) { return (n + to - 1) / to * to; }

// byte offsets of several buffers inside one allocation; -1: none
struct Layout {
  long long size = 0;
  long long add(long long bytes) {
    const long long at = size;
    size += pad(bytes, 256);
    return at;
  }
  // room for the operand image of a matrix, or none where it is read as it is
  static bool direct(const Tensor& t) {
    return t.scalar_type() != at::kFloat && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && pitch(t) % 8 == 0;
  }
  long long image(const Tensor& t) {
    if (direct(t)) return -1;
    return add(t.size(0) * pad(t.size(1), 16) * (t.scalar_type() == at::kFloat ? 6 : 2));
  }
};
void* at_offset(const Tensor& buf, long long offset) { return offset < 0 ? nullptr : static_cast<char*>(buf.data_ptr()) + offset; }

// Byte offsets of what the forward pass leaves in its workspace: images of the three operands, the hidden values and (training) G and U.
// The backward pass takes them from its node: which operands needed an image was decided by the tensors of the forward pass.
struct FfnBuffers {
  Layout layout;
  long long x = -1, w_in = -1, w_out = -1, h = -1, z = -1;
  FfnBuffers() = default;
  explicit FfnBuffers(const std::vector<int64_t>& kept) : x(kept[0]), w_in(kept[1]), w_out(kept[2]), h(kept[3]), z(kept[4]) {
    layout.size = kept[5];
  }
  std::vector<int64_t> keep() const { return {x, w_in, w_out, h, z, layout.size}; }
  FfnBuffers(const Tensor& x2, const Tensor& wi, const Tensor& wo, bool train, bool few) {
    const long long m = x2.size(0), f = pad(wo.size(1), 16), planes = x2.scalar_type() == at::kFloat ? 3 : 1;
    x = few ? -1 : layout.image(x2);
    w_in = few ? -1 : layout.image(wi);
    w_out = few ? -1 : layout.image(wo);
    h = layout.add(few ? 4 * m * f : planes * m * f * 2);
    z = train ? layout.add(2 * pad(m, 32) * f * 4) : -1;
  }
};
Tensor bytes(long long n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }

Tensor ffn_run(const Tensor& x, const Tensor& x2, const Tensor& wi, const Tensor& wo, int64_t act, bool train, Tensor* kept,
               FfnBuffers* at_kept) {
  const int m = (int)x2.size(0), d = (int)x2.size(1), f = (int)wo.size(1), n = (int)wo.size(0), dt = dtype_code(x.scalar_type());
  const bool few = !train && gated_ffn_few(m, d, f, n, dt);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = n;
  Tensor y = empty(shape, x), partial;
  if (m == 0) {
    *kept = bytes(0, x);
    return y;
  }
  const FfnBuffers at(x2, wi, wo, train, few);
  Tensor buf = bytes(at.layout.size, x);
  const long long floats = few ? 0 : gated_ffn_partial_floats(m, d, f, n, dt, 0);
  if (floats) partial = empty_floats(floats, x);
  *at_kept = at;
  FfnForwardCall c = {};
  c.x = x2.data_ptr(); c.ldx = pitch(x2); c.x_img = at_offset(buf, at.x);
  c.w_in = wi.data_ptr(); c.ld_in = pitch(wi); c.in_img = at_offset(buf, at.w_in);
  c.w_out = wo.data_ptr(); c.ld_out = pitch(wo); c.out_img = at_offset(buf, at.w_out);
  c.h = at_offset(buf, at.h);
  c.z = static_cast<float*>(at_offset(buf, at.z));
  c.partial = static_cast<float*>(ptr(partial));
  c.y = y.data_ptr();
  c.m = m; c.d = d; c.f = f; c.n = n; c.act = act; c.dt = dt; c.few = few;
  c.st = stream_of(x);
  check(gated_ffn_forward(&c), "gated_ffn_forward");
  g_launches += c.launches;
  *kept = buf;
  return y;
}

struct GatedFfnFn : torch::autograd::Function<GatedFfnFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_in, const Tensor& w_out, int64_t act) {
    const Tensor x2 = rows_of(x), wi = rows_of(w_in), wo = rows_of(w_out);
    Tensor buf;
    FfnBuffers at;
    Tensor y = ffn_run(x, x2, wi, wo, act, true, &buf, &at);
    ctx->save_for_backward({x2, wi, wo, buf});
    ctx->saved_data["act"] = act;
    ctx->saved_data["sizes"] = std::vector<int64_t>{x2.size(0), x2.size(1), wo.size(1), wo.size(0)};
    ctx->saved_data["buffers"] = at.keep();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second_derivative("gated_ffn");
    no_tangent("gated_ffn", {&grads[0]});
    const variable_list saved = ctx->get_saved_variables();
    const Tensor& dy = grads[0];
    const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
    const FfnBuffers at(ctx->saved_data["buffers"].toIntVector());
    const int m = (int)sizes[0], d = (int)sizes[1], f = (int)sizes[2], n = (int)sizes[3], dt = dtype_code(dy.scalar_type());
    check_saved(saved[0], {m, d}, dy.scalar_type(), dy.device(), "gated_ffn");
    check_saved(saved[1], {2 * f, d}, dy.scalar_type(), dy.device(), "gated_ffn");
    check_saved(saved[2], {n, f}, dy.scalar_type(), dy.device(), "gated_ffn");
    check_saved(saved[3], {at.layout.size}, at::kByte, dy.device(), "gated_ffn");
    const c10::OptionalDeviceGuard guard(dy.device());
    std::vector<int64_t> shape = dy.sizes().vec();
    shape.back() = d;
    Tensor dx, dwi, dwo;
    if (ctx->needs_input_grad(0)) dx = empty(shape, dy);
    if (ctx->needs_input_grad(1)) dwi = empty({2 * f, d}, dy);
    if (ctx->needs_input_grad(2)) dwo = empty({n, f}, dy);
    if (m == 0) {
      if (dwi.defined()) dwi.zero_();
      if (dwo.defined()) dwo.zero_();
      return {dx, dwi, dwo, Tensor()};
    }
    const Tensor x2 = rows_of(saved[0]), wi = rows_of(saved[1]), wo = rows_of(saved[2]), buf = workspace_of(saved[3]), dy2 = rows_of(dy);
    Layout scratch;
    // operands that the forward pass read as they were and that came back otherwise get an image now
    const long long dy_img = scratch.image(dy2), x_img = at.x < 0 ? scratch.image(x2) : -1, in_img = at.w_in < 0 ? scratch.image(wi) : -1,
                    out_img = at.w_out < 0 ? scratch.image(wo) : -1;
    const long long dz = scratch.add((dt == 0 ? 3 : 1) * 4LL * m * pad(f, 16));
    const long long floats = gated_ffn_partial_floats(m, d, f, n, dt, 1), partial = floats ? scratch.add(4 * floats) : -1;
    const Tensor s = bytes(scratch.size, dy);
    FfnBackwardCall c = {};
    c.x = x2.data_ptr(); c.ldx = pitch(x2); c.x_img = x_img >= 0 ? at_offset(s, x_img) : at_offset(buf, at.x);
    c.w_in = wi.data_ptr(); c.ld_in = pitch(wi); c.in_img = in_img >= 0 ? at_offset(s, in_img) : at_offset(buf, at.w_in);
    c.w_out = wo.data_ptr(); c.ld_out = pitch(wo); c.out_img = out_img >= 0 ? at_offset(s, out_img) : at_offset(buf, at.w_out);
    c.make = (x_img >= 0 ? 1 : 0) | (in_img >= 0 ? 2 : 0) | (out_img >= 0 ? 4 : 0);
    c.dy = dy2.data_ptr(); c.ldy = pitch(dy2); c.dy_img = at_offset(s, dy_img);
    c.h = at_offset(buf, at.h);
    c.z = static_cast<float*>(at_offset(buf, at.z));
    c.dz = at_offset(s, dz);
    c.partial = static_cast<float*>(at_offset(s, partial));
    c.dx = ptr(dx); c.dw_in = ptr(dwi); c.dw_out = ptr(dwo);
    c.m = m; c.d = d; c.f = f; c.n = n; c.act = ctx->saved_data["act"].toInt(); c.dt = dt;
    c.st = stream_of(dy);
    check(gated_ffn_backward(&c), "gated_ffn_backward");
    g_launches += c.launches;
    return {dx, dwi, dwo, Tensor()};
  }
};

bool gated_ffn_ok(const Tensor& x, const Tensor& w_in, const Tensor& w_out) {
  if (!(x.is_cuda() && dtype_code(x.scalar_type()) >= 0 && x.dim() >= 1 && w_in.dim() == 2 && w_out.dim() == 2)) return false;
  if (!(w_in.scalar_type() == x.scalar_type() && w_out.scalar_type() == x.scalar_type() && w_in.device() == x.device() &&
        w_out.device() == x.device()))
    return false;
  if (!(x.size(-1) == w_in.size(1) && w_in.size(0) == 2 * w_out.size(1) && w_in.size(0) > 0 && w_in.size(1) > 0 && w_out.size(0) > 0))
    return false;
  const int64_t most = 1 << 30;
  return x.numel() / x.size(-1) < most && w_in.size(0) < most && w_in.size(1) < most && w_out.size(0) < most;
}

Tensor gated_ffn(const Tensor& x, const Tensor& w_in, const Tensor& w_out, int64_t act) {
  if (!gated_ffn_ok(x, w_in, w_out))
    throw pybind11::value_error(
        "gated_ffn: needs x [..., D], w_in [2 F, D] and w_out [N, F] on one CUDA device and of one type (fp32, bf16 or fp16): got " +
        describe(x) + ", " + describe(w_in) + ", " + describe(w_out));
  no_tangent("gated_ffn", {&x, &w_in, &w_out});
  const c10::OptionalDeviceGuard guard(x.device());
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w_in) || wants_grad(w_out)))
    return GatedFfnFn::apply(x, w_in, w_out, act);
  Tensor buf;
  FfnBuffers at;
  return ffn_run(x, rows_of(x), rows_of(w_in), rows_of(w_out), act, false, &buf, &at);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  // wrapped: an allocation that fails raises PyTorch's own exception
  m.def("layer_norm", torch::wrap_pybind_function(layer_norm));
  m.def("layer_norm_supported", [](const Tensor& x, const Maybe& weight, const Maybe& bias) {
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    return layer_norm_ok(x, w, b) && !has_tangent(x) && !has_tangent(w) && !has_tangent(b);
  });
  m.def("dropout", torch::wrap_pybind_function(dropout));
  m.def("gated_ffn", torch::wrap_pybind_function(gated_ffn));
  m.def("gated_ffn_supported", [](const Tensor& x, const Tensor& w_in, const Tensor& w_out) {
    return gated_ffn_ok(x, w_in, w_out) && !has_tangent(x) && !has_tangent(w_in) && !has_tangent(w_out);
  });
  m.def("has_tangent", &has_tangent);
  m.def("launches", []() { return g_launches.load(); });
}
