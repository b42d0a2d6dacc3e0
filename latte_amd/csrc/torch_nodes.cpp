// The autograd nodes of linear and rms_norm (latte_amd/dense.py) over the C entry points of include/latte_hip.h.
//
// Host time is what small layers cost: as Python Functions a forward and backward took about 120 us of it, most in
// interpreter code on two threads that hand the interpreter lock to each other; the device needs 20 to 40 us for the same.
// The entry points come from the library that latte_amd._lib has loaded (init), so this module links none of them.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include "../../include/latte_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Entry {
  decltype(&lt_last_error) last_error;
  decltype(&lt_mx8_quantize) mx8_quantize;
  decltype(&lt_mx8_dequantize) mx8_dequantize;
  decltype(&lt_linear_mx8_workspace_bytes) linear_mx8_ws;
  decltype(&lt_linear_mx8_fwd) linear_mx8;
  decltype(&lt_linear_workspace_bytes) linear_ws;
  decltype(&lt_linear_fwd) linear_fwd;
  decltype(&lt_linear_bwd_workspace_bytes) linear_bwd_ws;
  decltype(&lt_linear_bwd) linear_bwd;
  decltype(&lt_rms_norm_fwd) rms_fwd;
  decltype(&lt_rms_norm_bwd_workspace_bytes) rms_bwd_ws;
  decltype(&lt_rms_norm_bwd) rms_bwd;
  decltype(&lt_bn_workspace_bytes) bn_ws;
  decltype(&lt_bn_stats) bn_stats;
  decltype(&lt_bn_apply_mx8) bn_apply;
  decltype(&lt_bn_bwd_reduce_mx8) bn_reduce;
  decltype(&lt_bn_bwd_apply_mx8) bn_bwd;
} lt;

void check(const char* name, int rc) {
  if (rc == 0) return;
  const char* m = lt.last_error();
  TORCH_CHECK(false, name, " failed (rc=", rc, "): ", m ? m : "");
}

int dtype_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return LT_DT_F32;
    case at::kBFloat16: return LT_DT_BF16;
    case at::kHalf: return LT_DT_F16;
    default: TORCH_CHECK_TYPE(false, name, ": expected float32, bfloat16 or float16, got ", t.dtype());
  }
}

// `t` checked against the operand it goes with: type, device, shape
void like(const Tensor& t, const Tensor& ref, at::IntArrayRef shape, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == ref.scalar_type(), name, ": expected ", ref.dtype(), ", got ", t.dtype());
  TORCH_CHECK_VALUE(t.device() == ref.device(), name, ": on ", t.device(), ", the other operands on ", ref.device());
  TORCH_CHECK_VALUE(t.sizes() == shape, name, ": expected shape ", shape, ", got ", t.sizes());
}

// the C entry points take row lengths and output widths as 32-bit numbers
bool fits32(int64_t n) { return n >= 1 && n < INT32_MAX; }

// the kernels read memory as it lies: the lazy minus sign of a view (the imaginary part of a conjugate) is carried out first
Tensor plain(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor dense(const Tensor& t) { return plain(t).contiguous(); }

// a 2-D tensor with neighbouring columns and its row stride: a view wherever the strides allow one
struct Rows {
  Tensor t;
  int64_t n = 0, ld = 0;
  Rows() = default;
  Rows(const Tensor& x, int64_t cols) {
    if (!x.defined()) return;
    t = x.dim() == 2 ? plain(x) : plain(x).reshape({-1, cols});
    if (t.stride(1) != 1 && cols > 1) t = t.contiguous();
    n = t.size(0);
    ld = n > 1 ? t.stride(0) : cols;   // a single row's stride means nothing
  }
  void* p() const { return t.defined() ? t.data_ptr() : nullptr; }
};

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// the current stream of the tensor's own device, whatever device is current
lt_stream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
// the shape of a result: x's with the last extent n.  Results are made in it: a view made inside a node could not be
// changed in place afterwards
std::vector<int64_t> last(const Tensor& x, int64_t n) {
  std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
  s.back() = n;
  return s;
}
// workspace of one call: torch's allocator (and a graph's private pool) keeps it from any other stream or graph
Tensor workspace(int64_t bytes, const Tensor& like) { return at::empty({bytes > 256 ? bytes : 256}, like.options().dtype(at::kByte)); }

// Forward-mode tangents would be lost without a word: the kernels see values only.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
void no_tangents(std::initializer_list<Tensor> ts) {
  for (const auto& t : ts)
    TORCH_CHECK(!has_tangent(t), "forward-mode derivatives are not implemented for the dense operators (forward_ad.unpack_dual gives the value)");
}

// A captured backward pass that goes on into a graph made before the capture on the default stream makes that stream wait for the
// capturing one as well (any other stream joins the capture).  Only the pass itself knows which gradients it was asked for.
void not_into_eager(const Tensor& dy) {
  const c10::DeviceGuard on(dy.device());
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  const c10::StreamId def = c10::hip::getDefaultHIPStream(dy.get_device()).id();
  for (size_t i = 0; i < node->num_outputs(); ++i) {
    if (!node->task_should_compute_output(i)) continue;
    const auto stream = node->next_edge(i).function->stream();
    TORCH_CHECK(!stream || stream->id() != def, "this backward pass can not be captured: it goes on into a graph that was made on the "
                "default stream before the capture; compute that part within the capture, or detach it");
  }
}

void no_second(const char* name, const variable_list& grads) {
  // a backward pass runs with gradients enabled only where its own graph is asked for, which these kernels do not build
  TORCH_CHECK(!at::GradMode::is_enabled(), name, ": gradients of gradients are not implemented (create_graph=True)");
  for (const auto& g : grads) no_tangents({g});
  for (const auto& g : grads)
    if (g.defined()) return not_into_eager(g);
}

// x held in mx8: e4m3 values and a scale byte per 32 neighbours
std::pair<Tensor, Tensor> quantize(const Rows& x, int64_t K, int dt) {
  Tensor q = at::empty({x.n, K}, x.t.options().dtype(at::kFloat8_e4m3fn)), s = at::empty({x.n, (K + 31) / 32}, x.t.options().dtype(at::kByte));
  check("lt_mx8_quantize", lt.mx8_quantize(x.p(), x.ld, x.n, (int32_t)K, dt, q.data_ptr(), s.data_ptr(), stream_of(x.t)));
  return {q, s};
}

enum { NEED_X = 1, NEED_W = 2, NEED_B = 4, NEED_R = 8 };
int64_t needs(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& r) {
  no_tangents({x, w, b, r});
  if (!at::GradMode::is_enabled()) return 0;
  auto need = [](const Tensor& t) { return t.defined() && t.requires_grad(); };
  const int64_t n = (need(x) ? NEED_X : 0) | (need(w) ? NEED_W : 0) | (need(b) ? NEED_B : 0) | (need(r) ? NEED_R : 0);
  if (!n) return 0;
  // While an eager graph of a leaf lives, the leaf's gradient is accumulated on that graph's stream.  A captured backward
  // pass would make that stream wait for the capturing one, which ends the capture and the process with it.  (Inputs that
  // were themselves computed before the capture: not_into_eager.)
  const c10::DeviceGuard on(x.device());
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) {
    const c10::StreamId here = c10::hip::getCurrentHIPStream(x.get_device()).id();   // the same id under torch's device name
    for (const Tensor* t : {&x, &w, &b, &r}) {
      if (!need(*t) || !t->is_leaf()) continue;
      const auto acc = torch::autograd::impl::try_get_grad_accumulator(*t);
      const auto stream = acc ? acc->stream() : std::optional<c10::Stream>();
      TORCH_CHECK(!stream || stream->id() == here, "a backward pass of this leaf can not be captured: a graph made on another stream still holds it; "
                  "let go of that graph's results first");
    }
  }
  return n;
}

// which of these this backward pass was asked for (autograd.grad of some of the inputs).  A node's edges are its tensors that exist,
// in the order of its arguments.
int64_t asked(const AutogradContext* ctx, int64_t need, bool has_b) {
  int64_t n = 0;
  if ((need & NEED_X) && ctx->needs_input_grad(0)) n |= NEED_X;
  if ((need & NEED_W) && ctx->needs_input_grad(1)) n |= NEED_W;
  if ((need & NEED_B) && ctx->needs_input_grad(2)) n |= NEED_B;
  if ((need & NEED_R) && ctx->needs_input_grad(has_b ? 3 : 2)) n |= NEED_R;
  return n;
}

// ------------------------------------------------------------------ linear
struct LinearSaved {
  Tensor x, scales, w, deriv;
  std::vector<int64_t> meta;   // K, N, deriv kind, row strides of x and w, needs, a bias or none, then the shape of x
};

Tensor linear_forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& r, int64_t act, bool mx8, int64_t need,
                      LinearSaved* keep) {
  const c10::DeviceGuard on(x.device());   // a null stream is the current device's
  const int dt = dtype_of(x, "linear x");
  const int64_t N = w.size(0), K = w.size(1);
  const Rows x2(x, K), w2(w, K), r2(r, N);
  const Tensor bias = b.defined() ? dense(b) : b;
  const int64_t M = x2.n;
  int kind = LT_DERIV_NONE;
  if (act != LT_ACT_NONE && (need & (NEED_X | NEED_W | NEED_B))) kind = act == LT_ACT_RELU ? LT_DERIV_BITS : mx8 ? LT_DERIV_BYTE : LT_DERIV_FULL;
  Tensor y = at::empty(last(x, N), x.options()), deriv;
  if (kind == LT_DERIV_BITS) deriv = at::empty({M, (N + 15) / 16}, x.options().dtype(at::kShort));
  else if (kind == LT_DERIV_BYTE) deriv = at::empty({M, N}, x.options().dtype(at::kByte));
  else if (kind == LT_DERIV_FULL) deriv = at::empty({M, N}, x.options().dtype(dt == LT_DT_F32 ? at::kFloat : at::kShort));
  const int64_t wsb = lt.linear_ws(M, (int32_t)K, (int32_t)N, dt);
  const Tensor ws = wsb > 0 ? workspace(wsb, x) : Tensor();
  check("lt_linear_fwd", lt.linear_fwd(x2.p(), x2.ld, w2.p(), w2.ld, ptr(bias), r2.p(), r2.ld, (int32_t)act, M, (int32_t)K, (int32_t)N, dt,
                                       y.data_ptr(), ptr(deriv), kind, ptr(ws), wsb, stream_of(x)));
  if (keep) {
    int64_t ldx = x2.ld;
    if (need & NEED_W) {
      if (mx8) {
        std::tie(keep->x, keep->scales) = quantize(x2, K, dt);
        ldx = K;
      } else {
        keep->x = x2.t;
      }
    }
    if (need & NEED_X) keep->w = w2.t;
    keep->deriv = deriv;
    keep->meta = {K, N, kind, ldx, w2.ld, need, b.defined()};
    for (auto s : x.sizes()) keep->meta.push_back(s);
  }
  return y;
}

struct LinearNode : public torch::autograd::Function<LinearNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& b,
                        const std::optional<Tensor>& r, int64_t act, bool mx8, int64_t need) {
    LinearSaved keep;
    Tensor y = linear_forward(x, w, b.value_or(Tensor()), r.value_or(Tensor()), act, mx8, need, &keep);
    ctx->save_for_backward({keep.x, keep.scales, keep.w, keep.deriv});
    ctx->saved_data["meta"] = keep.meta;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second("linear", grads);
    const c10::DeviceGuard on(grads[0].device());
    const auto saved = ctx->get_saved_variables();
    const auto meta = ctx->saved_data["meta"].toIntVector();
    const int64_t K = meta[0], N = meta[1], need = asked(ctx, meta[5], meta[6]);
    const Tensor& dy = grads[0];
    Tensor dx, dw, db;
    if (need & (NEED_X | NEED_W | NEED_B)) {
      const Rows g(dy, N);
      const int dt = dtype_of(dy, "linear");
      if (need & NEED_X) dx = at::empty({g.n, K}, dy.options());
      if (need & NEED_W) dw = at::empty({N, K}, dy.options());
      if (need & NEED_B) db = at::empty({N}, dy.options());
      const Tensor ws = workspace(lt.linear_bwd_ws(g.n, (int32_t)K, (int32_t)N, dt, saved[1].defined()), dy);
      check("lt_linear_bwd",
            lt.linear_bwd(g.p(), g.ld, ptr(saved[0]), meta[3], ptr(saved[1]), ptr(saved[2]), meta[4], ptr(saved[3]), (int32_t)meta[2], g.n,
                          (int32_t)K, (int32_t)N, dt, ptr(dx), ptr(dw), ptr(db), ws.data_ptr(), ws.numel(), stream_of(dy)));
      if (dx.defined() && meta.size() != 9) dx = dx.view(at::IntArrayRef(meta.data() + 7, meta.size() - 7));
    }
    return {dx, dw, db, need & NEED_R ? dy : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor linear(const Tensor& x, const Tensor& w, const std::optional<Tensor>& b_, const std::optional<Tensor>& r_, int64_t act, bool mx8) {
  const Tensor b = b_.value_or(Tensor()), r = r_.value_or(Tensor());
  dtype_of(x, "linear x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && x.size(-1) == w.size(1) && fits32(w.size(0)) && fits32(w.size(1)), "linear: x ",
                    x.sizes(), " and weight ", w.sizes(), " do not go together");
  like(w, x, w.sizes(), "linear weight");
  if (b.defined()) like(b, x, {w.size(0)}, "linear bias");
  if (r.defined()) {
    like(r, x, last(x, w.size(0)), "linear residual");
  }
  const int64_t need = needs(x, w, b, r);
  if (!need) return linear_forward(x, w, b, r, act, mx8, 0, nullptr);
  return LinearNode::apply(x, w, b_, r_, act, mx8, need);
}

// ------------------------------------------------------------------ rms_norm
struct RmsSaved {
  Tensor h, h2, h8, h8s, w, rstd;
  int64_t ldh = 0, ldh2 = 0;
};

std::pair<Tensor, Tensor> rms_forward(const Tensor& x, const Tensor& w_, const Tensor& r, double eps, bool mx8, RmsSaved* keep) {
  const c10::DeviceGuard on(x.device());
  const int dt = dtype_of(x, "rms_norm x");
  const int64_t C = x.size(-1);
  const Rows x2(x, C), r2(r, C);
  const Tensor w = dense(w_);
  Tensor y = at::empty(x.sizes(), x.options()), h, h8, h8s, rstd;
  if (r.defined()) h = at::empty(x.sizes(), x.options());
  if (keep) {
    rstd = at::empty({x2.n}, x.options().dtype(at::kFloat));
    if (mx8) {
      h8 = at::empty({x2.n, C}, x.options().dtype(at::kFloat8_e4m3fn));
      h8s = at::empty({x2.n, (C + 31) / 32}, x.options().dtype(at::kByte));
    }
  }
  check("lt_rms_norm_fwd", lt.rms_fwd(x2.p(), x2.ld, r2.p(), r2.ld, w.data_ptr(), (float)eps, x2.n, (int32_t)C, dt, ptr(h), y.data_ptr(), nullptr,
                                      nullptr, ptr(h8), ptr(h8s), (float*)ptr(rstd), stream_of(x)));
  if (keep) {
    if (!mx8) {   // h: x itself without a residual, the stored sum in fp32, the two summands beside 16-bit types
      const bool sum = r.defined() && dt == LT_DT_F32;
      keep->h = sum ? h : x2.t;
      keep->ldh = sum ? C : x2.ld;
      if (r.defined() && !sum) keep->h2 = r2.t, keep->ldh2 = r2.ld;
    }
    keep->h8 = h8;
    keep->h8s = h8s;
    keep->w = w;
    keep->rstd = rstd;
  }
  return {y, h};
}

struct RmsNode : public torch::autograd::Function<RmsNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const std::optional<Tensor>& r, double eps, bool mx8,
                               int64_t need) {
    RmsSaved keep;
    auto [y, h] = rms_forward(x, w, r.value_or(Tensor()), eps, mx8, &keep);
    ctx->save_for_backward({keep.h, keep.h8, keep.h8s, keep.w, keep.rstd, keep.h2});
    std::vector<int64_t> meta = {keep.ldh, need, keep.ldh2};
    for (auto s : x.sizes()) meta.push_back(s);
    ctx->saved_data["meta"] = meta;
    ctx->set_materialize_grads(false);   // a sum that nothing reads costs no zeros
    if (h.defined()) return {y, h};
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second("rms_norm", grads);
    const auto saved = ctx->get_saved_variables();
    const auto meta = ctx->saved_data["meta"].toIntVector();
    const int64_t need = asked(ctx, meta[1], false);
    const Tensor &w = saved[3], &rstd = saved[4];
    const Tensor dy = grads[0], dh = grads.size() > 1 ? grads[1] : Tensor();
    Tensor dx, dw;
    if (!dy.defined()) {   // only the sum was used: its gradient passes through
      if (dh.defined() && (need & NEED_W)) dw = at::zeros_like(w);
      return {need & NEED_X ? dh : Tensor(), dw, need & NEED_R ? dh : Tensor(), Tensor(), Tensor(), Tensor()};
    }
    const c10::DeviceGuard on(dy.device());
    const int64_t C = w.size(0), M = rstd.size(0);
    const Rows g(dy, C), gh(dh, C);
    if (need & (NEED_X | NEED_R)) dx = at::empty({M, C}, dy.options());
    if (need & NEED_W) dw = at::empty({C}, dy.options());
    const int64_t wsb = dw.defined() ? lt.rms_bwd_ws(M, (int32_t)C) : 0;
    const Tensor ws = dw.defined() ? workspace(wsb, dy) : Tensor();
    check("lt_rms_norm_bwd", lt.rms_bwd(g.p(), g.ld, gh.p(), gh.ld, ptr(saved[0]), meta[0], ptr(saved[5]), meta[2], ptr(saved[1]), ptr(saved[2]), w.data_ptr(),
                                        (const float*)rstd.data_ptr(), M, (int32_t)C, dtype_of(dy, "rms_norm"), ptr(dx), ptr(dw), ptr(ws),
                                        ws.defined() ? ws.numel() : 0, stream_of(dy)));
    if (dx.defined() && meta.size() != 5) dx = dx.view(at::IntArrayRef(meta.data() + 3, meta.size() - 3));
    return {need & NEED_X ? dx : Tensor(), dw, need & NEED_R ? dx : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

int check_rms(const Tensor& x, const Tensor& w, const Tensor& r) {
  const int dt = dtype_of(x, "rms_norm x");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 16384, "rms_norm: expected rows of 1 to 16384 elements, got shape ", x.sizes());
  like(w, x, {x.size(-1)}, "rms_norm weight");
  if (r.defined()) like(r, x, x.sizes(), "rms_norm residual");
  return dt;
}

variable_list rms_norm(const Tensor& x, const Tensor& w, const std::optional<Tensor>& r_, double eps, bool mx8) {
  const Tensor r = r_.value_or(Tensor());
  check_rms(x, w, r);
  const int64_t need = needs(x, w, Tensor(), r);
  if (!need) {
    auto [y, h] = rms_forward(x, w, r, eps, false, nullptr);
    if (h.defined()) return {y, h};
    return {y};
  }
  return RmsNode::apply(x, w, r_, eps, mx8, need);
}

// ------------------------------------------------------------------ batch_norm with 8-bit checkpoints (fp32, batch statistics)
void bn_like(const Tensor& t, const Tensor& x, at::IntArrayRef shape, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, name, ": expected torch.float32, got ", t.dtype());
  like(t, x, shape, name);
}

struct BnNode : public torch::autograd::Function<BnNode> {
  // -> y, mean, var
  static variable_list forward(AutogradContext* ctx, const Tensor& x_, const Tensor& gamma_, const Tensor& beta_, const std::optional<Tensor>& r_,
                               double eps, bool relu, bool post, int64_t need) {
    const c10::DeviceGuard on(x_.device());
    const Tensor x = dense(x_), gamma = dense(gamma_), beta = dense(beta_);
    const Tensor r = r_ ? dense(*r_) : Tensor();
    const int64_t V = x.size(0);
    const int32_t C = (int32_t)x.size(1);
    const lt_stream_t stream = stream_of(x);
    Tensor y = at::empty_like(x), mean = at::empty({C}, x.options()), var = at::empty({C}, x.options());
    Tensor q = at::empty({V, C}, x.options().dtype(at::kFloat8_e4m3fn)), s = at::empty({V, (C + 31) / 32}, x.options().dtype(at::kByte)), mask;
    if (relu) mask = at::empty({V, (C + 15) / 16}, x.options().dtype(at::kShort));
    const Tensor ws = workspace(lt.bn_ws(V, C), x);
    check("lt_bn_stats", lt.bn_stats(x.data_ptr<float>(), V, C, ws.data_ptr(), ws.numel(), mean.data_ptr<float>(), var.data_ptr<float>(), stream));
    check("lt_bn_apply_mx8", lt.bn_apply(x.data_ptr<float>(), mean.data_ptr<float>(), var.data_ptr<float>(), gamma.data_ptr<float>(),
                                         beta.data_ptr<float>(), (float)eps, (const float*)ptr(r), post ? 3 : relu ? 1 : 0, y.data_ptr<float>(),
                                         q.data_ptr(), s.data_ptr(), ptr(mask), V, C, stream));
    ctx->save_for_backward({q, s, mask, mean, var, gamma});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["meta"] = std::vector<int64_t>{need, post};
    ctx->mark_non_differentiable({mean, var});
    ctx->set_materialize_grads(false);   // the statistics' gradients are never there: no zeros for them
    return {y, mean, var};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    no_second("batch_norm", grads);
    if (!grads[0].defined()) return variable_list(8);
    const auto saved = ctx->get_saved_variables();
    const auto meta = ctx->saved_data["meta"].toIntVector();
    const float eps = (float)ctx->saved_data["eps"].toDouble();
    const int64_t need = asked(ctx, meta[0], true);
    const bool post = meta[1] != 0;
    const c10::DeviceGuard on(grads[0].device());
    const Tensor dy = dense(grads[0]);
    const Tensor &q = saved[0], &s = saved[1], &mask = saved[2], &mean = saved[3], &var = saved[4], &gamma = saved[5];
    const int64_t V = q.size(0);
    const int32_t C = (int32_t)q.size(1);
    const lt_stream_t stream = stream_of(dy);
    Tensor dgamma, dbeta, dx, dr;
    if (need & NEED_X) dx = at::empty_like(dy);
    if ((need & NEED_R) && !post) dr = at::empty_like(dy);
    const bool sums = need & (NEED_X | NEED_W | NEED_B);   // the residual's gradient needs none
    if (sums || dr.defined()) dgamma = at::empty({C}, dy.options()), dbeta = at::empty({C}, dy.options());
    if (sums) {
      const Tensor ws = workspace(lt.bn_ws(V, C), dy);
      check("lt_bn_bwd_reduce_mx8", lt.bn_reduce(dy.data_ptr<float>(), q.data_ptr(), s.data_ptr(), ptr(mask), mean.data_ptr<float>(),
                                                 var.data_ptr<float>(), eps, V, C, ws.data_ptr(), ws.numel(), dbeta.data_ptr<float>(),
                                                 dgamma.data_ptr<float>(), stream));
    }
    if (dx.defined() || dr.defined())
      check("lt_bn_bwd_apply_mx8",
            lt.bn_bwd(dy.data_ptr<float>(), q.data_ptr(), s.data_ptr(), ptr(mask), mean.data_ptr<float>(), var.data_ptr<float>(),
                      gamma.data_ptr<float>(), eps, dbeta.data_ptr<float>(), dgamma.data_ptr<float>(), (float*)ptr(dx), (float*)ptr(dr), V, C, stream));
    if ((need & NEED_R) && post) dr = dy;   // the residual bypasses the ReLU
    return {dx, need & NEED_W ? dgamma : Tensor(), need & NEED_B ? dbeta : Tensor(), dr, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

variable_list batch_norm_mx8(const Tensor& x, const Tensor& gamma, const Tensor& beta, const std::optional<Tensor>& r, double eps, bool relu,
                             bool post) {
  TORCH_CHECK_VALUE(x.dim() == 2 && fits32(x.size(1)), "batch_norm: expected a [rows, channels] matrix, got shape ", x.sizes());
  bn_like(x, x, x.sizes(), "batch_norm x");
  bn_like(gamma, x, {x.size(1)}, "batch_norm gamma");
  bn_like(beta, x, {x.size(1)}, "batch_norm beta");
  if (r) bn_like(*r, x, x.sizes(), "batch_norm residual");
  return BnNode::apply(x, gamma, beta, r, eps, relu, post && relu && r, needs(x, gamma, beta, r.value_or(Tensor())));
}

// ------------------------------------------------------------------ mx8 (no gradients)
std::pair<Tensor, Tensor> quantize_mx8(const Tensor& x) {
  const int dt = dtype_of(x, "quantize_mx8");
  TORCH_CHECK_VALUE(x.dim() >= 1 && fits32(x.size(-1)), "quantize_mx8: expected rows of 1 to 2^31 - 2 elements, got shape ", x.sizes());
  at::NoGradGuard off;
  const c10::DeviceGuard on(x.device());
  return quantize(Rows(x, x.size(-1)), x.size(-1), dt);
}

Tensor dequantize_mx8(const Tensor& q, const Tensor& s, at::ScalarType dtype) {
  TORCH_CHECK_VALUE(fits32(q.size(1)), "Mx8.dequantize: expected rows of 1 to 2^31 - 2 elements, got shape ", q.sizes());
  const c10::DeviceGuard on(q.device());
  Tensor out = at::empty(q.sizes(), q.options().dtype(dtype));
  check("lt_mx8_dequantize", lt.mx8_dequantize(q.data_ptr(), s.data_ptr(), q.size(0), (int32_t)q.size(1), dtype_of(out, "Mx8.dequantize"),
                                               out.data_ptr(), stream_of(q)));
  return out;
}

void no_gradient(const char* what, std::initializer_list<Tensor> ts) {
  no_tangents(ts);
  for (const auto& t : ts)
    TORCH_CHECK(!(at::GradMode::is_enabled() && t.defined() && t.requires_grad()), what, "; call it under torch.no_grad()");
}

Tensor linear_mx8(const Tensor& x, const Tensor& xs, const Tensor& w, const Tensor& ws_, const std::optional<Tensor>& b_,
                  const std::optional<Tensor>& r_, int64_t act, std::optional<at::ScalarType> dtype) {
  const Tensor b = b_.value_or(Tensor()), r = r_.value_or(Tensor());
  no_gradient("linear: mx8 operands carry no gradient", {b, r});
  const c10::DeviceGuard on(x.device());
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
  TORCH_CHECK_VALUE(w.size(1) == K && fits32(K) && fits32(N), "linear: x ", x.sizes(), " and weight ", w.sizes(), " do not go together");
  TORCH_CHECK_VALUE(w.device() == x.device(), "linear weight: on ", w.device(), ", the other operands on ", x.device());
  const at::ScalarType out = dtype ? *dtype : b.defined() ? b.scalar_type() : r.defined() ? r.scalar_type() : at::kBFloat16;
  TORCH_CHECK_TYPE(out == at::kBFloat16 || out == at::kHalf, "linear: results of mx8 operands are bfloat16 or float16, not ", out);
  Tensor y = at::empty({M, N}, x.options().dtype(out));
  if (b.defined()) like(b, y, {N}, "linear bias");
  if (r.defined()) like(r, y, {M, N}, "linear residual");
  const Tensor bias = b.defined() ? dense(b) : b;
  const Rows r2(r, N);
  const int64_t wsb = lt.linear_mx8_ws(M, (int32_t)K, (int32_t)N);
  const Tensor ws = wsb > 0 ? workspace(wsb, x) : Tensor();
  check("lt_linear_mx8_fwd", lt.linear_mx8(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws_.data_ptr(), ptr(bias), r2.p(), r2.ld, (int32_t)act, M,
                                           (int32_t)K, (int32_t)N, dtype_of(y, "linear"), y.data_ptr(), ptr(ws), wsb, stream_of(x)));
  return y;
}

// -> values, scales of y (and h)
variable_list rms_norm_mx8(const Tensor& x, const Tensor& w, const std::optional<Tensor>& r_, double eps) {
  const Tensor r = r_.value_or(Tensor());
  const int dt = check_rms(x, w, r);
  no_gradient("rms_norm: out='mx8' carries no gradient", {x, w, r});
  const c10::DeviceGuard on(x.device());
  const int64_t C = x.size(-1);
  const Rows x2(x, C), r2(r, C);
  Tensor q = at::empty({x2.n, C}, x.options().dtype(at::kFloat8_e4m3fn)), s = at::empty({x2.n, (C + 31) / 32}, x.options().dtype(at::kByte)), h;
  if (r.defined()) h = at::empty(x.sizes(), x.options());
  check("lt_rms_norm_fwd", lt.rms_fwd(x2.p(), x2.ld, r2.p(), r2.ld, dense(w).data_ptr(), (float)eps, x2.n, (int32_t)C, dt, ptr(h), nullptr,
                                      q.data_ptr(), s.data_ptr(), nullptr, nullptr, nullptr, stream_of(x)));
  if (h.defined()) return {q, s, h};
  return {q, s};
}

template <class F>
void bind(F& f, const py::dict& d, const char* name) { f = reinterpret_cast<F>(d[name].cast<uintptr_t>()); }

void init(const py::dict& d) {
  bind(lt.last_error, d, "lt_last_error");
  bind(lt.mx8_quantize, d, "lt_mx8_quantize");
  bind(lt.mx8_dequantize, d, "lt_mx8_dequantize");
  bind(lt.linear_mx8_ws, d, "lt_linear_mx8_workspace_bytes");
  bind(lt.linear_mx8, d, "lt_linear_mx8_fwd");
  bind(lt.linear_ws, d, "lt_linear_workspace_bytes");
  bind(lt.linear_fwd, d, "lt_linear_fwd");
  bind(lt.linear_bwd_ws, d, "lt_linear_bwd_workspace_bytes");
  bind(lt.linear_bwd, d, "lt_linear_bwd");
  bind(lt.rms_fwd, d, "lt_rms_norm_fwd");
  bind(lt.rms_bwd_ws, d, "lt_rms_norm_bwd_workspace_bytes");
  bind(lt.rms_bwd, d, "lt_rms_norm_bwd");
  bind(lt.bn_ws, d, "lt_bn_workspace_bytes");
  bind(lt.bn_stats, d, "lt_bn_stats");
  bind(lt.bn_apply, d, "lt_bn_apply_mx8");
  bind(lt.bn_reduce, d, "lt_bn_bwd_reduce_mx8");
  bind(lt.bn_bwd, d, "lt_bn_bwd_apply_mx8");
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("init", &init, "entry points of liblatte_hip.so by name (addresses)");
  m.def("linear", &linear, py::call_guard<py::gil_scoped_release>());
  m.def("rms_norm", &rms_norm, py::call_guard<py::gil_scoped_release>());
  m.def("batch_norm_mx8", &batch_norm_mx8, py::call_guard<py::gil_scoped_release>());
  m.def("quantize_mx8", &quantize_mx8, py::call_guard<py::gil_scoped_release>());
  m.def("dequantize_mx8", &dequantize_mx8, py::call_guard<py::gil_scoped_release>());
  m.def("linear_mx8", &linear_mx8, py::call_guard<py::gil_scoped_release>());
  m.def("rms_norm_mx8", &rms_norm_mx8, py::call_guard<py::gil_scoped_release>());
}
