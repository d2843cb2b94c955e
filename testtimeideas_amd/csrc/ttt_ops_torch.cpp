// ttt_ops_torch.cpp — torch binding of the operators at the model's tail
// (include/ttt_ops.h): layer norm and linear cross entropy as autograd
// functions whose backward is differentiable under create_graph=True, in C++
// so that neither pass enters the interpreter (see AttnBwd in ttt_torch.cpp).
//
// Outputs, statistics and workspaces come from torch's caching allocator on
// the operands' device, calls go to torch's current stream of that device, and
// a nonzero status raises RuntimeError with the library's message.  Operands
// the C ABI does not take (a column stride, rows out of alignment) are copied.
// No kernel runs here and nothing falls back.
#include <torch/extension.h>
#include <torch/csrc/autograd/custom_function.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cstring>
#include <utility>
#include <vector>

#include "../../include/ttt_ops.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> OptTensor;

int32_t dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return TTT_F16;
    case at::kBFloat16: return TTT_BF16;
    case at::kFloat: return TTT_F32;
    default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t.scalar_type(), "; expected float16, bfloat16 or float32");
  }
  return -1;
}

void check(int rc, const char* what) {
  TORCH_CHECK(rc == 0, what, " failed (status ", rc, "): ", ttt_last_error());
}

// The current device and the stream to launch on, for the operands' device.
struct Launch {
  c10::DeviceGuard guard;
  c10::DeviceIndex index;
  explicit Launch(const Tensor& t) : guard(t.device()), index(t.device().index()) {}
  void* stream() const { return static_cast<void*>(c10::hip::getCurrentHIPStream(index).stream()); }
};

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

// `t` [..., d] as [n, d] with contiguous columns; align: 16-byte rows.
Tensor as_rows(const Tensor& t, bool align) {
  const int64_t d = t.size(-1);
  Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / std::max<int64_t>(d, 1), d});
  const int64_t eb = r.element_size(), st = r.size(0) > 1 ? r.stride(0) : d;
  bool ok = (r.stride(1) == 1 || d <= 1) && st >= d && st <= (1 << 22);
  if (align) ok = ok && reinterpret_cast<uintptr_t>(r.data_ptr()) % 16 == 0 && (st * eb) % 16 == 0;
  return ok ? r : at::empty({r.size(0), d}, r.options()).copy_(r);
}

ttt_rows rows_of(const Tensor& t) {
  ttt_rows r;
  r.data = ptr(t);
  r.stride = !t.defined() ? 0 : t.size(0) > 1 ? t.stride(0) : t.size(1);
  return r;
}

Tensor bytes(int64_t n, const Tensor& like) {
  return n > 0 ? at::empty({n}, like.options().dtype(at::kByte)) : Tensor();
}

OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }
Tensor tensor_of(const OptTensor& t) { return t ? *t : Tensor(); }

// A second derivative's result as a function of what it was formed from,
// whose own derivative raises.  (torch's DelayedError hangs on nothing: where
// another path leads to the leaves, as through dy, its error is left out of
// the walk and the third derivative would silently lack these terms.)
struct Once : public torch::autograd::Function<Once> {
  static Tensor forward(AutogradContext*, const Tensor& t, const OptTensor&, const OptTensor&, const OptTensor&,
                        const OptTensor&, const OptTensor&, const OptTensor&) {
    return t.detach();
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "trying to differentiate twice a function that was marked with @once_differentiable");
    return {};
  }
};

// out as functions of from (at most six) where a graph is being recorded.
variable_list once(variable_list out, const variable_list& from) {
  if (!at::GradMode::is_enabled()) return out;
  OptTensor f[6];
  for (size_t i = 0; i < from.size() && i < 6; ++i) f[i] = opt(from[i]);
  for (Tensor& t : out)
    if (t.defined()) t = Once::apply(t, f[0], f[1], f[2], f[3], f[4], f[5]);
  return out;
}

// Refuses a backward pass that is being captured while an eager graph of one of
// its leaves is alive.  The leaf's gradient node is then of the eager graph's
// stream; the engine makes that stream wait for the captured one, the capture
// ends with work that never joins it, and the process with it.
void check_capture(std::initializer_list<Tensor> leaves) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  for (const Tensor& t : leaves) {
    if (!t.defined() || !t.is_leaf() || !t.requires_grad()) continue;
    const std::shared_ptr<torch::autograd::Node> node = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!node) continue;
    const auto stream = node->stream();
    TORCH_CHECK(!stream || *stream == c10::impl::VirtualGuardImpl(t.device().type()).getStream(t.device()),
                "a backward pass cannot be captured while a graph of the same leaf tensor, recorded on another "
                "stream, is alive: drop that graph (the tensors computed from the leaf) before the capture");
  }
}

Tensor as_type(const Tensor& t, const Tensor& like) {
  return !t.defined() || t.scalar_type() == like.scalar_type() ? t : t.to(like.scalar_type());
}

// ---------------------------------------------------------------------------
// Layer norm over the last dimension.
// ---------------------------------------------------------------------------
ttt_norm_problem norm_problem(const Tensor& x, const Tensor& w, double eps) {
  ttt_norm_problem p;
  p.dtype = dtype_code(x);
  p.param_dtype = w.defined() ? dtype_code(w) : p.dtype;
  p.rows = x.size(0);
  p.cols = x.size(1);
  p.eps = static_cast<float>(eps);
  return p;
}

// w or b, whichever is given: the parameters' type.
const Tensor& either(const Tensor& w, const Tensor& b) { return w.defined() ? w : b; }

Tensor packed(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

// y (and mean, rstd with `stats`)
std::vector<Tensor> norm_fwd(const Tensor& x_, const Tensor& w_, const Tensor& b_, double eps, bool stats) {
  const Launch on(x_);
  Tensor y = at::empty(x_.sizes(), x_.options());
  const Tensor x = as_rows(x_, false), w = packed(w_), b = packed(b_);
  Tensor mean, rstd;
  if (stats) {
    mean = at::empty({x.size(0)}, x.options().dtype(at::kFloat));
    rstd = at::empty({x.size(0)}, x.options().dtype(at::kFloat));
  }
  if (x.numel() == 0) return {y, mean, rstd};
  const ttt_norm_problem p = norm_problem(x, either(w, b), eps);
  ttt_rows rx = rows_of(x), ry;
  ry.data = y.data_ptr();
  ry.stride = x.size(1);
  check(ttt_norm_fwd(&p, &rx, ptr(w), ptr(b), &ry, fptr(mean), fptr(rstd), on.stream()), "ttt_norm_fwd");
  return {y, mean, rstd};
}

// dx, dw, db: those asked for.  like: a tensor of the parameters' type.
std::vector<Tensor> norm_bwd(const Tensor& dy_, const Tensor& x_, const Tensor& w_, const Tensor& mean,
                             const Tensor& rstd, at::ScalarType ptype, double eps, bool nx, bool nw, bool nb) {
  const Launch on(x_);
  const Tensor x = as_rows(x_, false), dy = as_rows(dy_, false), w = packed(w_);
  const auto po = x.options().dtype(ptype);
  Tensor dx, dw, db;
  if (nx) dx = at::empty(x_.sizes(), x_.options());
  if (nw) dw = at::empty({x.size(1)}, po);
  if (nb) db = at::empty({x.size(1)}, po);
  if (x.numel() == 0) {
    if (nw) dw.zero_();
    if (nb) db.zero_();
    return {dx, dw, db};
  }
  ttt_norm_problem p = norm_problem(x, w, eps);
  p.param_dtype = ptype == at::kFloat ? TTT_F32 : p.dtype;
  const int64_t n = nw || nb ? ttt_norm_workspace_size(&p) : 0;
  TORCH_CHECK(n >= 0, "ttt_norm_workspace_size failed: ", ttt_last_error());
  const Tensor ws = bytes(n, x);
  const ttt_rows rx = rows_of(x), rdy = rows_of(dy);
  ttt_rows rdx;
  rdx.data = ptr(dx);
  rdx.stride = x.size(1);
  check(ttt_norm_bwd(&p, &rx, ptr(w), &rdy, fptr(mean), fptr(rstd), &rdx, ptr(dw), ptr(db), ptr(ws), n, on.stream()),
        "ttt_norm_bwd");
  return {dx, dw, db};
}

struct NormBwd : public torch::autograd::Function<NormBwd> {
  static variable_list forward(AutogradContext* ctx, const Tensor& dy, const Tensor& x, const OptTensor& w_,
                               const Tensor& mean, const Tensor& rstd, int64_t ptype, double eps, bool nx, bool nw,
                               bool nb) {
    const Tensor w = tensor_of(w_);
    const std::vector<Tensor> r =
        norm_bwd(dy, x, w, mean, rstd, static_cast<at::ScalarType>(ptype), eps, nx, nw, nb);
    ctx->save_for_backward({dy, x, w, mean, rstd});
    ctx->saved_data["ptype"] = ptype;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["have"] = static_cast<int64_t>(nx) | static_cast<int64_t>(nw) << 1 | static_cast<int64_t>(nb) << 2;
    ctx->set_materialize_grads(false);
    variable_list out;
    for (const Tensor& t : r)
      if (t.defined()) out.push_back(t);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const int64_t have = ctx->saved_data["have"].toInt();
    const auto ptype = static_cast<at::ScalarType>(ctx->saved_data["ptype"].toInt());
    variable_list out(10);
    const variable_list s = ctx->get_saved_variables();
    {
      at::NoGradGuard no_grad;
      Tensor c[3];
      size_t n = 0;
      for (int i = 0; i < 3; ++i)
        if (have >> i & 1) c[i] = g[n++];
      if (!c[0].defined() && !c[1].defined() && !c[2].defined()) return out;
      const Launch on(s[1]);
      check_capture({s[0], s[1], s[2]});
      const Tensor x = as_rows(s[1], false), dy = as_rows(s[0], false), w = packed(s[2]);
      Tensor a;
      if (c[0].defined()) a = as_rows(as_type(c[0], x), false);
      for (int i = 1; i < 3; ++i)
        if (c[i].defined()) c[i] = c[i].to(ptype).contiguous();
      Tensor gdy, gx, gw;
      if (ctx->needs_input_grad(0)) gdy = at::empty(s[0].sizes(), s[0].options());
      if (ctx->needs_input_grad(1)) gx = at::empty(s[1].sizes(), s[1].options());
      if (s[2].defined() && ctx->needs_input_grad(2)) gw = at::empty(s[2].sizes(), s[2].options());
      if (x.numel() == 0) {
        if (gw.defined()) gw.zero_();
      } else {
        ttt_norm_problem p = norm_problem(x, w, ctx->saved_data["eps"].toDouble());
        p.param_dtype = ptype == at::kFloat ? TTT_F32 : p.dtype;
        const int64_t nb = gw.defined() ? ttt_norm_workspace_size(&p) : 0;
        TORCH_CHECK(nb >= 0, "ttt_norm_workspace_size failed: ", ttt_last_error());
        const Tensor ws = bytes(nb, x);
        const ttt_rows rx = rows_of(x), rdy = rows_of(dy), ra = rows_of(a);
        ttt_rows rgx, rgdy;
        rgx.data = ptr(gx);
        rgdy.data = ptr(gdy);
        rgx.stride = rgdy.stride = x.size(1);
        check(ttt_norm_gg(&p, &rx, ptr(w), &rdy, fptr(s[3]), fptr(s[4]), &ra, ptr(c[1]), ptr(c[2]), &rgx, ptr(gw),
                          &rgdy, ptr(ws), nb, on.stream()),
              "ttt_norm_gg");
      }
      out[0] = gdy;
      out[1] = gx;
      out[2] = gw;
    }
    variable_list from{s[0], s[1], s[2]};
    from.insert(from.end(), g.begin(), g.end());
    return once(std::move(out), from);
  }
};

struct Norm : public torch::autograd::Function<Norm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& w_, const OptTensor& b_, double eps) {
    const Tensor w = tensor_of(w_), b = tensor_of(b_);
    const std::vector<Tensor> r = norm_fwd(x, w, b, eps, true);
    const Tensor& p = either(w, b);
    ctx->save_for_backward({x, w, r[1], r[2]});
    ctx->saved_data["ptype"] = static_cast<int64_t>(p.defined() ? p.scalar_type() : x.scalar_type());
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["given"] = static_cast<int64_t>(w.defined()) | static_cast<int64_t>(b.defined()) << 1;
    return r[0];
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    const int64_t given = ctx->saved_data["given"].toInt(), ptype = ctx->saved_data["ptype"].toInt();
    const double eps = ctx->saved_data["eps"].toDouble();
    const bool nx = ctx->needs_input_grad(0), nw = (given & 1) && ctx->needs_input_grad(1),
               nb = (given & 2) && ctx->needs_input_grad(2);
    variable_list out(4);
    if (!nx && !nw && !nb) return out;
    check_capture({s[0], s[1]});
    const Tensor dy = as_type(g[0], s[0]);
    variable_list r;
    if (at::GradMode::is_enabled()) {
      r = NormBwd::apply(dy, s[0], opt(s[1]), s[2], s[3], ptype, eps, nx, nw, nb);
    } else {
      for (const Tensor& t : norm_bwd(dy, s[0], s[1], s[2], s[3], static_cast<at::ScalarType>(ptype), eps, nx, nw, nb))
        if (t.defined()) r.push_back(t);
    }
    size_t n = 0;
    if (nx) out[0] = r[n++];
    if (nw) out[1] = r[n++];
    if (nb) out[2] = r[n++];
    return out;
  }
};

bool wants_grad(std::initializer_list<Tensor> ts) {
  return at::GradMode::is_enabled() &&
         std::any_of(ts.begin(), ts.end(), [](const Tensor& t) { return t.defined() && t.requires_grad(); });
}

Tensor layer_norm(const Tensor& x, const OptTensor& w_, const OptTensor& b_, double eps) {
  const Tensor w = tensor_of(w_), b = tensor_of(b_);
  if (wants_grad({x, w, b})) return Norm::apply(x, opt(w), opt(b), eps);
  return norm_fwd(x, w, b, eps, false)[0];
}

// ---------------------------------------------------------------------------
// Linear cross entropy.
// ---------------------------------------------------------------------------
ttt_lce_problem lce_problem(const Tensor& x, const Tensor& w, int64_t reduction, int64_t ignore) {
  ttt_lce_problem p;
  p.dtype = dtype_code(x);
  p.reduction = static_cast<int32_t>(reduction);
  p.rows = x.size(0);
  p.cols = x.size(1);
  p.vocab = w.size(0);
  p.ignore_index = ignore;
  return p;
}

Tensor lce_rows(const Tensor& t) { return as_rows(t, t.scalar_type() != at::kFloat && t.size(-1) % 8 == 0); }

Tensor lce_workspace(const ttt_lce_problem& p, int32_t entry, const Tensor& like, int64_t* n) {
  *n = ttt_lce_workspace_size(&p, entry);
  TORCH_CHECK(*n >= 0, "ttt_lce_workspace_size failed: ", ttt_last_error());
  return bytes(*n, like);
}

// loss, row_stats
std::vector<Tensor> lce_fwd(const Tensor& x_, const Tensor& w_, const Tensor& target, const Tensor& mask,
                            int64_t reduction, int64_t ignore) {
  const Launch on(x_);
  const Tensor x = lce_rows(x_), w = lce_rows(w_);
  const auto fo = x.options().dtype(at::kFloat);
  const int64_t n = x.size(0);
  Tensor loss = reduction == TTT_REDUCE_NONE ? at::empty(target.sizes(), fo) : at::empty({}, fo);
  Tensor stats = at::empty({2 * n + 2}, fo);
  if (n == 0) {
    if (reduction != TTT_REDUCE_NONE) loss.zero_();
    return {loss, stats};
  }
  const ttt_lce_problem p = lce_problem(x, w, reduction, ignore);
  int64_t nb;
  const Tensor ws = lce_workspace(p, TTT_LCE_FWD, x, &nb);
  const ttt_rows rx = rows_of(x), rw = rows_of(w);
  check(ttt_lce_fwd(&p, &rx, &rw, target.data_ptr<int64_t>(), fptr(mask), fptr(loss), fptr(stats), ptr(ws), nb,
                    on.stream()),
        "ttt_lce_fwd");
  return {loss, stats};
}

// dx, dw: those asked for; and dx32 with `keep`.
std::vector<Tensor> lce_bwd(const Tensor& g, const Tensor& x_, const Tensor& w_, const Tensor& target,
                            const Tensor& mask, const Tensor& stats, int64_t reduction, int64_t ignore, bool nx,
                            bool nw, bool keep) {
  const Launch on(x_);
  const Tensor x = lce_rows(x_), w = lce_rows(w_);
  Tensor dx, dw, dx32;
  if (nx) dx = at::empty(x_.sizes(), x_.options());
  if (nx && keep) dx32 = at::empty(x_.sizes(), x_.options().dtype(at::kFloat));
  if (nw) dw = at::empty(w_.sizes(), w_.options());
  if (x.size(0) == 0) {
    if (nw) dw.zero_();
    return {dx, dw, dx32};
  }
  const ttt_lce_problem p = lce_problem(x, w, reduction, ignore);
  int64_t nb;
  const Tensor ws = lce_workspace(p, TTT_LCE_BWD, x, &nb);
  const ttt_rows rx = rows_of(x), rw = rows_of(w);
  ttt_rows rdx, rdw;
  rdx.data = ptr(dx);
  rdw.data = ptr(dw);
  rdx.stride = rdw.stride = x.size(1);
  check(ttt_lce_bwd(&p, &rx, &rw, target.data_ptr<int64_t>(), fptr(mask), fptr(stats), fptr(g), &rdx, &rdw,
                    fptr(dx32), ptr(ws), nb, on.stream()),
        "ttt_lce_bwd");
  return {dx, dw, dx32};
}

struct LceBwd : public torch::autograd::Function<LceBwd> {
  static variable_list forward(AutogradContext* ctx, const Tensor& g, const Tensor& x, const Tensor& w,
                               const Tensor& target, const OptTensor& mask_, const Tensor& stats, int64_t reduction,
                               int64_t ignore, bool nx, bool nw) {
    const Tensor mask = tensor_of(mask_);
    const std::vector<Tensor> r = lce_bwd(g, x, w, target, mask, stats, reduction, ignore, nx, nw, true);
    ctx->save_for_backward({g, x, w, target, mask, stats, r[2]});
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["nx"] = nx;
    ctx->saved_data["nw"] = nw;
    ctx->set_materialize_grads(false);
    variable_list out;
    if (nx) out.push_back(r[0]);
    if (nw) out.push_back(r[1]);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    variable_list out(10);
    const variable_list s = ctx->get_saved_variables();
    {
      at::NoGradGuard no_grad;
      const bool nx = ctx->saved_data["nx"].toBool(), nw = ctx->saved_data["nw"].toBool();
      Tensor a = nx ? g[0] : Tensor(), b = nw ? g[nx ? 1 : 0] : Tensor();
      if (!a.defined() && !b.defined()) return out;
      const Launch on(s[1]);
      check_capture({s[0], s[1], s[2]});
      const Tensor x = lce_rows(s[1]), w = lce_rows(s[2]);
      if (a.defined()) a = lce_rows(as_type(a, x));
      if (b.defined()) b = lce_rows(as_type(b, x));
      Tensor gg, gx, gw;
      if (ctx->needs_input_grad(0)) gg = at::empty(s[0].sizes(), s[0].options());
      if (ctx->needs_input_grad(1)) gx = at::empty(s[1].sizes(), s[1].options());
      if (ctx->needs_input_grad(2)) gw = at::empty(s[2].sizes(), s[2].options());
      if (x.size(0) == 0) {
        if (gw.defined()) gw.zero_();
        if (gg.defined()) gg.zero_();
      } else {
        const ttt_lce_problem p =
            lce_problem(x, w, ctx->saved_data["reduction"].toInt(), ctx->saved_data["ignore"].toInt());
        int64_t nb;
        const Tensor ws = lce_workspace(p, TTT_LCE_GG, x, &nb);
        const ttt_rows rx = rows_of(x), rw = rows_of(w), ra = rows_of(a), rb = rows_of(b);
        ttt_rows rgx, rgw;
        rgx.data = ptr(gx);
        rgw.data = ptr(gw);
        rgx.stride = rgw.stride = x.size(1);
        check(ttt_lce_gg(&p, &rx, &rw, s[3].data_ptr<int64_t>(), fptr(s[4]), fptr(s[5]), fptr(s[0]), fptr(s[6]), &ra,
                         &rb, &rgx, &rgw, fptr(gg), ptr(ws), nb, on.stream()),
              "ttt_lce_gg");
      }
      out[0] = gg;
      out[1] = gx;
      out[2] = gw;
    }
    variable_list from{s[0], s[1], s[2]};
    from.insert(from.end(), g.begin(), g.end());
    return once(std::move(out), from);
  }
};

struct Lce : public torch::autograd::Function<Lce> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& target,
                        const OptTensor& mask_, int64_t reduction, int64_t ignore) {
    const Tensor mask = tensor_of(mask_);
    const std::vector<Tensor> r = lce_fwd(x, w, target, mask, reduction, ignore);
    ctx->save_for_backward({x, w, target, mask, r[1]});
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["ignore"] = ignore;
    return r[0];
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    const int64_t reduction = ctx->saved_data["reduction"].toInt(), ignore = ctx->saved_data["ignore"].toInt();
    const bool nx = ctx->needs_input_grad(0), nw = ctx->needs_input_grad(1);
    variable_list out(6);
    if (!nx && !nw) return out;
    check_capture({s[0], s[1]});
    Tensor go = g[0];
    if (go.scalar_type() != at::kFloat) go = go.to(at::kFloat);
    go = go.contiguous();
    variable_list r;
    if (at::GradMode::is_enabled()) {
      r = LceBwd::apply(go, s[0], s[1], s[2], opt(s[3]), s[4], reduction, ignore, nx, nw);
    } else {
      const std::vector<Tensor> d = lce_bwd(go, s[0], s[1], s[2], s[3], s[4], reduction, ignore, nx, nw, false);
      if (nx) r.push_back(d[0]);
      if (nw) r.push_back(d[1]);
    }
    size_t n = 0;
    if (nx) out[0] = r[n++];
    if (nw) out[1] = r[n++];
    return out;
  }
};

// target (int64) and mask (fp32) contiguous, of hidden's leading shape.
Tensor linear_cross_entropy(const Tensor& x, const Tensor& w, const Tensor& target, const OptTensor& mask_,
                            int64_t reduction, int64_t ignore) {
  const Tensor mask = tensor_of(mask_);
  if (wants_grad({x, w})) return Lce::apply(x, w, target, opt(mask), reduction, ignore);
  return lce_fwd(x, w, target, mask, reduction, ignore)[0];
}

}  // namespace

void bind_ops(py::module_& m) {
  m.def("layer_norm", &layer_norm, "layer norm over the last dimension, twice differentiable");
  m.def("linear_cross_entropy", &linear_cross_entropy,
        "softmax cross entropy of hidden @ weight^T, twice differentiable");
}
