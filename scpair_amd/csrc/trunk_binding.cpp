// Autograd nodes of the residual-trunk operators (scpair_amd/ops.py: gated_residual_norm, pack8, unpack8, act8, linear8).
//
// A step of a trunk is many short calls, and what bounds a call of minibatch size is the host: a Python backward runs in the
// autograd engine's thread with cold caches and the interpreter's lock to hand over (1024 x 900 fp32, forward + backward of
// gated_residual_norm: 164 us in Python, of which the GPU works 32).  So these nodes are C++; arguments arrive checked and laid
// out by the Python functions, and every launch goes through the C ABI of libscpair_hip.so (include/scpair_hip.h).
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include "scpair_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Opt;

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

void check(int rc, const char* what) {
  if (rc == 0) return;
  TORCH_CHECK_VALUE(rc != -1 && rc != -2, what, ": ", scp_last_error());
  TORCH_CHECK(false, what, ": error ", rc, ": ", scp_last_error());
}

template <typename T = void>
T* ptr(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }
Tensor value(const Opt& t) { return t.has_value() ? *t : Tensor(); }
bool is16(const Tensor& t) { return t.scalar_type() == at::kBFloat16; }
Tensor fresh(const Tensor& like, at::IntArrayRef shape, at::ScalarType type) { return at::empty(shape, like.options().dtype(type)); }

// 2-D [rows, cols] with contiguous columns (a copy only if its strides are others)
Tensor rows_of(const Tensor& t) { return t.stride(1) == 1 || t.size(1) == 1 ? t : t.contiguous(); }

// Gradients of a node whose own derivative does not exist: asking for it raises instead of passing for a constant.
variable_list once(variable_list grads, const char* who) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list given;
  for (const Tensor& g : grads)
    if (g.defined()) given.push_back(g.set_requires_grad(true));
  auto node = std::make_shared<torch::autograd::DelayedError>(std::string(who) + ": a second derivative is not implemented",
                                                              (int64_t)given.size());
  given = (*node)(std::move(given));
  size_t i = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = given[i++];
  return grads;
}

// A call that needs no backward pass makes no node, and a launch is nothing that torch sees: a forward-mode tangent would get lost,
// and a trace would keep the call's result as a constant.  Both are refused, whether a node is made or not.
void visible(const char* who, std::initializer_list<const Tensor*> given) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), who, ": cannot be traced");
  for (const Tensor* t : given)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), who, ": forward-mode derivatives are not implemented");
}

// Which forward arguments want a gradient: absent tensors have no edge, so edges are counted along.
struct Needs {
  AutogradContext* ctx;
  size_t edge = 0;
  explicit Needs(AutogradContext* c) : ctx(c) {}
  bool operator()(bool present) { return present && ctx->needs_input_grad(edge++); }
};

// ---- 8-bit checkpoints ----------------------------------------------------------------------------------------------
std::pair<Tensor, Tensor> empty_packed(const Tensor& like, int64_t rows, int64_t cols) {
  const int64_t groups = (cols + 63) / 64;
  return {fresh(like, {rows, 64 * groups}, at::kChar), fresh(like, {rows, groups}, at::kByte)};
}

std::pair<Tensor, Tensor> pack8(const Tensor& x) {
  visible("pack8", {});
  c10::DeviceGuard guard(x.device());
  auto p = empty_packed(x, x.size(0), x.size(1));
  check(scp_pack8(ptr(x), is16(x), x.stride(0), x.size(0), (int)x.size(1), ptr<int8_t>(p.first), ptr<uint8_t>(p.second),
                  stream_of(x)), "scp_pack8");
  return p;
}

Tensor unpack8(const Tensor& codes, const Tensor& steps, int64_t cols, bool bf16) {
  visible("unpack8", {});
  c10::DeviceGuard guard(codes.device());
  Tensor out = fresh(codes, {codes.size(0), cols}, bf16 ? at::kBFloat16 : at::kFloat);
  check(scp_unpack8(ptr<int8_t>(codes), ptr<uint8_t>(steps), codes.size(0), (int)cols, ptr(out), bf16, stream_of(codes)),
        "scp_unpack8");
  return out;
}

// ---- act8 -----------------------------------------------------------------------------------------------------------
Tensor act8_forward(const Tensor& z, int64_t kind, double slope, Tensor* codes, Tensor* steps) {
  c10::DeviceGuard guard(z.device());
  Tensor out = fresh(z, z.sizes(), z.scalar_type());
  if (codes) std::tie(*codes, *steps) = empty_packed(z, z.size(0), z.size(1));
  check(scp_act8_fwd(ptr(z), is16(z), z.stride(0), z.size(0), (int)z.size(1), (int)kind, (float)slope, ptr(out),
                     codes ? ptr<int8_t>(*codes) : nullptr, steps ? ptr<uint8_t>(*steps) : nullptr, stream_of(z)), "scp_act8_fwd");
  return out;
}

struct Act8 : torch::autograd::Function<Act8> {
  static Tensor forward(AutogradContext* ctx, const Tensor& z, int64_t kind, double slope) {
    Tensor codes, steps, out = act8_forward(z, kind, slope, &codes, &steps);
    ctx->save_for_backward({codes, steps});
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["slope"] = slope;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor d = rows_of(grads[0]);
    c10::DeviceGuard guard(d.device());
    Tensor dz = fresh(d, d.sizes(), d.scalar_type());
    check(scp_act8_bwd(ptr<int8_t>(saved[0]), ptr<uint8_t>(saved[1]), d.size(0), (int)d.size(1), (int)ctx->saved_data["kind"].toInt(),
                       (float)ctx->saved_data["slope"].toDouble(), ptr(d), is16(d), d.stride(0), ptr(dz), stream_of(d)),
          "scp_act8_bwd");
    return once({dz, Tensor(), Tensor()}, "act8");
  }
};

Tensor act8(const Tensor& z, int64_t kind, double slope) {
  visible("act8", {&z});
  if (at::GradMode::is_enabled() && z.requires_grad()) return Act8::apply(z, kind, slope);
  return act8_forward(z, kind, slope, nullptr, nullptr);
}

// ---- linear8 --------------------------------------------------------------------------------------------------------
Tensor workspace(const Tensor& like, long bytes, const char* what) {
  if (bytes < 0) check(-1, what);
  return bytes ? fresh(like, {bytes}, at::kByte) : Tensor();
}

Tensor linear8_forward(const Tensor& x, const Tensor& W, const Tensor& b, bool split, Tensor* codes, Tensor* steps) {
  c10::DeviceGuard guard(x.device());
  const int64_t M = x.size(0), K = x.size(1), N = W.size(0);
  Tensor y = fresh(x, {M, N}, x.scalar_type());
  if (codes) std::tie(*codes, *steps) = empty_packed(x, M, K);
  if (M == 0) return y;
  ScpLinear8 a = {};
  a.x = ptr(x); a.W = ptr(W); a.b = ptr<float>(b); a.y = ptr(y);
  if (codes) a.codes = ptr<int8_t>(*codes), a.steps = ptr<uint8_t>(*steps);
  a.M = M; a.N = (int)N; a.K = (int)K; a.ldx = x.stride(0);
  a.x_bf16 = is16(x); a.w_bf16 = is16(W); a.ns = split ? 3 : 1;
  const Tensor ws = workspace(x, scp_linear8_fwd_ws(&a), "scp_linear8_fwd");
  a.ws = ptr(ws);
  check(scp_linear8_fwd(&a, stream_of(x)), "scp_linear8_fwd");
  return y;
}

struct Linear8 : torch::autograd::Function<Linear8> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& W, const Opt& b, bool split, bool keep) {
    Tensor codes, steps, y = linear8_forward(x, W, value(b), split, keep ? &codes : nullptr, keep ? &steps : nullptr);
    if (keep) ctx->save_for_backward({W, codes, steps});
    else ctx->save_for_backward({W});
    ctx->saved_data["cfg"] = (int64_t)(split + 2 * b.has_value());
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor W = saved[0].contiguous(), dy = rows_of(grads[0]);
    c10::DeviceGuard guard(dy.device());
    const int64_t cfg = ctx->saved_data["cfg"].toInt(), M = dy.size(0), N = W.size(0), K = W.size(1);
    Needs need(ctx);
    Tensor dx, dW, db;
    if (need(true)) dx = fresh(dy, {M, K}, dy.scalar_type());
    if (need(true)) dW = fresh(W, {N, K}, W.scalar_type());
    if (need(cfg & 2)) db = fresh(dy, {N}, at::kFloat);
    if (M == 0) {
      if (dW.defined()) dW.zero_();
      if (db.defined()) db.zero_();
    } else {
      ScpLinear8 a = {};
      a.W = ptr(W); a.dy = ptr(dy); a.dx = ptr(dx); a.dW = ptr(dW); a.db = ptr<float>(db);
      if (dW.defined()) a.codes = ptr<int8_t>(saved[1]), a.steps = ptr<uint8_t>(saved[2]);
      a.M = M; a.N = (int)N; a.K = (int)K; a.lddy = dy.stride(0);
      a.x_bf16 = is16(dy); a.w_bf16 = is16(W); a.ns = cfg & 1 ? 3 : 1;
      const Tensor ws = workspace(dy, scp_linear8_bwd_ws(&a), "scp_linear8_bwd");
      a.ws = ptr(ws);
      check(scp_linear8_bwd(&a, stream_of(dy)), "scp_linear8_bwd");
    }
    return once({dx, dW, db, Tensor(), Tensor()}, "linear8");
  }
};

Tensor linear8(const Tensor& x, const Tensor& W, const Opt& b, bool split) {
  const Tensor bias = value(b);
  visible("linear8", {&x, &W, &bias});
  if (at::GradMode::is_enabled() && (x.requires_grad() || W.requires_grad() || (b.has_value() && b->requires_grad())))
    return Linear8::apply(x, W, b, split, W.requires_grad());
  return linear8_forward(x, W, bias, split, nullptr, nullptr);
}

// ---- gated_residual_norm ----------------------------------------------------------------------------------------------
struct NormForm {
  int64_t post, pre, gate_mode, gate_act, scale_mode;
  double scale_value, eps;
  bool y16;
};

ScpResidualNorm norm_block(const variable_list& t, const NormForm& f) {
  ScpResidualNorm a = {};
  a.x = ptr(t[0]); a.h = ptr(t[1]); a.gate = ptr(t[2]); a.scale = ptr<float>(t[3]);
  a.w1 = ptr<float>(t[4]); a.b1 = ptr<float>(t[5]); a.w2 = ptr<float>(t[6]); a.b2 = ptr<float>(t[7]);
  a.rows = t[0].size(0); a.cols = (int)t[0].size(1);
  a.ldx = t[0].stride(0);
  if (t[1].defined()) a.ldh = t[1].stride(0);
  if (f.gate_mode == 1) a.ldg = t[2].stride(0);
  a.x_bf16 = is16(t[0]); a.h_bf16 = f.y16;
  a.post = (int)f.post; a.pre = (int)f.pre; a.gate_mode = (int)f.gate_mode; a.gate_act = (int)f.gate_act;
  a.scale_mode = (int)f.scale_mode; a.scale_value = (float)f.scale_value; a.eps = (float)f.eps;
  return a;
}

// r (undefined without a block), y; stats where asked for
std::pair<Tensor, Tensor> norm_forward(const variable_list& t, const NormForm& f, Tensor* stats) {
  c10::DeviceGuard guard(t[0].device());
  Tensor r, y = fresh(t[0], t[0].sizes(), f.y16 ? at::kBFloat16 : at::kFloat);
  if (t[1].defined()) r = fresh(t[0], t[0].sizes(), t[0].scalar_type());
  if (stats) *stats = fresh(t[0], {t[0].size(0), 4}, at::kFloat);
  if (t[0].size(0) == 0) return {r, y};
  ScpResidualNorm a = norm_block(t, f);
  a.r = ptr(r); a.y = ptr(y);
  if (stats) a.stats = ptr<float>(*stats);
  check(scp_residual_norm_fwd(&a, stream_of(t[0])), "scp_residual_norm_fwd");
  return {r, y};
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Opt& h, const Opt& gate, const Opt& scale, const Opt& w1,
                               const Opt& b1, const Opt& w2, const Opt& b2, const NormForm& f) {
    const variable_list t = {x, value(h), value(gate), value(scale), value(w1), value(b1), value(w2), value(b2)};
    Tensor stats;
    auto ry = norm_forward(t, f, &stats);
    variable_list keep = {stats};
    int64_t present = 0;
    for (int i = 0; i < 8; i++)
      if (t[i].defined()) {
        present |= 1 << i;
        keep.push_back(t[i]);
      }
    ctx->save_for_backward(std::move(keep));
    ctx->saved_data["form"] = std::vector<int64_t>{f.post, f.pre, f.gate_mode, f.gate_act, f.scale_mode, f.y16, present};
    ctx->saved_data["eps"] = std::vector<double>{f.scale_value, f.eps};
    ctx->set_materialize_grads(false);
    return ry.first.defined() ? variable_list{ry.first, ry.second} : variable_list{ry.second};
  }

  static variable_list backward(AutogradContext* ctx, variable_list up) {
    const Tensor dr0 = up.size() == 2 ? up[0] : Tensor(), dy0 = up.back();
    variable_list out(9);
    if (!dr0.defined() && !dy0.defined()) return out;
    const std::vector<int64_t> c = ctx->saved_data["form"].toIntVector();
    const std::vector<double> v = ctx->saved_data["eps"].toDoubleVector();
    const NormForm f = {c[0], c[1], c[2], c[3], c[4], v[0], v[1], c[5] != 0};
    const variable_list saved = ctx->get_saved_variables();
    variable_list t(8);
    for (int i = 0, j = 1; i < 8; i++)
      if (c[6] >> i & 1) t[i] = saved[j++];
    const Tensor& x = t[0];
    c10::DeviceGuard guard(x.device());
    const int64_t rows = x.size(0), cols = x.size(1);
    Needs need(ctx);
    bool want[8];
    int columns = 0;
    for (int i = 0; i < 8; i++) {
      want[i] = need(t[i].defined());
      columns += want[i] && (i > 3 || (i == 3 && f.scale_mode == 2) || (i == 2 && f.gate_mode == 3));
    }
    if (want[0]) out[0] = fresh(x, {rows, cols}, x.scalar_type());
    if (want[1]) out[1] = fresh(x, {rows, cols}, t[1].scalar_type());
    // the gradients of one number a column: rows of one small tensor, each from a 256-byte boundary
    const int64_t pitch = (cols + 63) / 64 * 64;
    const Tensor small = columns ? fresh(x, {columns, pitch}, at::kFloat) : Tensor();
    int next = 0;
    for (int i = 2; i < 8; i++) {
      if (!want[i]) continue;
      if (i > 3 || (i == 3 && f.scale_mode == 2) || (i == 2 && f.gate_mode == 3)) out[i] = small.as_strided({cols}, {1}, pitch * next++);
      else out[i] = fresh(x, t[i].sizes(), t[i].scalar_type());
    }
    if (rows == 0) {           // no cell: nothing to launch, the parameters' sums are empty
      for (Tensor& g : out)
        if (g.defined()) g.zero_();
      return once(std::move(out), "gated_residual_norm");
    }
    const Tensor dr = dr0.defined() ? rows_of(dr0) : dr0, dy = dy0.defined() ? rows_of(dy0) : dy0;
    ScpResidualNorm a = norm_block(t, f);
    a.stats = ptr<float>(saved[0]);
    a.dr = ptr(dr); a.dy = ptr(dy);
    if (dr.defined()) a.lddr = dr.stride(0);
    if (dy.defined()) a.lddy = dy.stride(0);
    a.dx = ptr(out[0]); a.dh = ptr(out[1]); a.dgate = ptr(out[2]);
    a.dscale = ptr<float>(out[3]); a.dw1 = ptr<float>(out[4]); a.db1 = ptr<float>(out[5]);
    a.dw2 = ptr<float>(out[6]); a.db2 = ptr<float>(out[7]);
    Tensor ws;
    if (columns || want[3]) ws = fresh(x, {scp_residual_norm_bwd_ws_floats(rows, (int)cols)}, at::kFloat);
    a.ws = ptr<float>(ws);
    check(scp_residual_norm_bwd(&a, stream_of(x)), "scp_residual_norm_bwd");
    return once(std::move(out), "gated_residual_norm");
  }
};

std::pair<Opt, Tensor> residual_norm(const Tensor& x, const Opt& h, const Opt& gate, const Opt& scale, const Opt& w1, const Opt& b1,
                                     const Opt& w2, const Opt& b2, int64_t post, int64_t pre, int64_t gate_mode, int64_t gate_act,
                                     int64_t scale_mode, double scale_value, double eps, bool y16) {
  const NormForm f = {post, pre, gate_mode, gate_act, scale_mode, scale_value, eps, y16};
  const variable_list t = {x, value(h), value(gate), value(scale), value(w1), value(b1), value(w2), value(b2)};
  visible("gated_residual_norm", {&t[0], &t[1], &t[2], &t[3], &t[4], &t[5], &t[6], &t[7]});
  bool track = false;
  if (at::GradMode::is_enabled())
    for (const Tensor& v : t) track = track || (v.defined() && v.requires_grad());
  if (!track) {
    auto ry = norm_forward(t, f, nullptr);
    return {ry.first.defined() ? Opt(ry.first) : std::nullopt, ry.second};
  }
  const variable_list o = ResidualNorm::apply(x, h, gate, scale, w1, b1, w2, b2, f);
  return {o.size() == 2 ? Opt(o[0]) : std::nullopt, o.back()};
}

}  // namespace

PYBIND11_MODULE(_trunk, m) {
  m.doc() = "autograd nodes of the residual-trunk operators; use scpair_amd.ops, which checks the arguments";
  m.def("pack8", &pack8);
  m.def("unpack8", &unpack8);
  m.def("act8", &act8);
  m.def("linear8", &linear8);
  m.def("residual_norm", &residual_norm);
}
