// The PyTorch side of what stands beside the chunked op: the element-wise gated recurrence and the norms around a block.  As in
// torch_ops.cpp, ops.py keeps the public functions and each of them is one call into this module.
#include "torch_util.h"

namespace lethe_torch {
namespace {

using torch::autograd::SavedVariable;

// First order only: a second derivative runs into the error node that wraps the gradients.
struct FirstOrderNode : public torch::autograd::Node {
  std::vector<SavedVariable> kept;
  bool released = false;

  virtual variable_list first_order(const variable_list& grads) = 0;

  void release_variables() override {
    for (auto& s : kept) s.reset_data();
    released = true;
  }
  variable_list apply(variable_list&& grads) override {
    bool second = false, any = false;
    for (const Tensor& t : grads) {
      any = any || t.defined();
      second = second || (torch::autograd::GradMode::is_enabled() && t.defined() && t.requires_grad());
    }
    variable_list out(num_outputs());
    if (!any) return out;
    {
      at::NoGradGuard no_grad;
      TORCH_CHECK(!released, torch::autograd::ERR_BACKWARD_TWICE);
      out = first_order(grads);
    }
    if (!second) return out;
    for (auto& t : out)
      if (t.defined()) t = t.detach().requires_grad_(true);
    auto err = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", static_cast<int64_t>(out.size()));
    return (*err)(std::move(out));
  }
  void keep(const Tensor& t, bool is_output = false) { kept.emplace_back(t, is_output); }
};

bool wants_grad(std::initializer_list<Tensor> ts) {
  if (!torch::autograd::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// a tensor that may be in 32 bits or in the type of the activations; anything else is read as fp32
Tensor in_type(const Tensor& t, at::ScalarType dt) {
  return t.scalar_type() == dt || t.scalar_type() == at::kFloat ? t : t.to(at::kFloat);
}

// stride between neighbours over dimensions [from, to) taken as one; -1: there is none
int64_t joint_stride(const Tensor& t, int64_t from, int64_t to) {
  int64_t stride = 0, want = 0;
  bool first = true;
  for (int64_t i = to - 1; i >= from; --i) {
    if (t.size(i) == 1) continue;
    if (first) stride = t.stride(i);
    else if (t.stride(i) != want) return -1;
    first = false;
    want = t.stride(i) * t.size(i);
  }
  return stride;
}

// ---------------------------------------------------------------------------------------------
// Element-wise gated recurrence
// ---------------------------------------------------------------------------------------------
// readable as [B, L, D] with strides for batch and token
Tensor tokens(const Tensor& t) { return lazy(t) || !packed_from(t, 2) ? as(t, t.scalar_type()) : t; }

LetheGdnDiagArgs diag_args(const Tensor& x, const Tensor& g, bool complement) {
  LetheGdnDiagArgs a;
  memset(&a, 0, sizeof(a));
  a.B = x.size(0); a.L = x.size(1); a.D = x.numel() / (a.B * a.L);
  a.x_type = code(x.scalar_type()); a.g_type = code(g.scalar_type()); a.complement = complement;
  a.x = ptr(x); a.x_batch = step_of(x, 0); a.x_token = step_of(x, 1);
  a.g = ptr(g); a.g_batch = step_of(g, 0); a.g_token = step_of(g, 1);
  a.status = status_word(x.device().index());
  return a;
}
Tensor diag_work(LetheGdnDiagArgs* a, const Tensor& like, bool backward) {
  a->work_bytes = lethe_gdn_diag_work_bytes(a->B, a->L, a->D, a->x_type, backward);
  Tensor w;
  if (a->work_bytes) {
    w = at::empty({static_cast<int64_t>(a->work_bytes)}, like.options().dtype(at::kByte));
    a->work = ptr(w);
  }
  return w;
}

struct DiagScanBackward : public FirstOrderNode {      // kept: x, g, states
  bool complement = false, empty = false;
  at::ScalarType g_type, h0_type;
  std::vector<int64_t> state_shape;
  std::string name() const override { return "DiagScanBackward"; }

  variable_list first_order(const variable_list& grads) override {
    auto self = getptr();
    const Tensor x = kept[0].unpack(self), g = kept[1].unpack(self);
    c10::cuda::CUDAGuard guard(x.device());
    const auto o32 = x.options().dtype(at::kFloat);
    const Tensor dhT = as32(grads[1]);
    Tensor dx, dg, dh0;
    if (task_should_compute_output(2)) dh0 = at::empty(state_shape, o32);
    if (empty) {
      if (task_should_compute_output(0)) dx = at::zeros(x.sizes(), x.options());
      if (task_should_compute_output(1)) dg = at::zeros(g.sizes(), g.options());
      if (dh0.defined()) dhT.defined() ? dh0.copy_(dhT) : dh0.zero_();
    } else {
      const Tensor states = kept[2].unpack(self), xt = tokens(x), gt = tokens(g);
      const Tensor d = grads[0].defined() ? tokens(grads[0].scalar_type() == x.scalar_type() ? grads[0] : grads[0].to(x.scalar_type())) : Tensor();
      LetheGdnDiagArgs a = diag_args(xt, gt, complement);
      const Tensor at_states = reinterpret_cast<uintptr_t>(states.data_ptr()) % 4 || !states.is_contiguous() ? states.clone() : states;
      a.states = ptr<float>(at_states);
      if (d.defined()) {
        a.d_h = ptr(d); a.d_h_batch = step_of(d, 0); a.d_h_token = step_of(d, 1);
      }
      a.dhT = ptr<float>(dhT);
      if (task_should_compute_output(0)) dx = at::empty(x.sizes(), x.options());
      if (task_should_compute_output(1)) dg = at::empty(g.sizes(), g.options());
      a.dx = ptr(dx); a.dg = ptr(dg); a.dh0 = ptr<float>(dh0);
      const Tensor work = diag_work(&a, x, true);
      check(lethe_gdn_diag_backward(&a, stream_of(x)));
    }
    return {dx, dg.defined() ? cast_back(dg, g_type) : dg, dh0.defined() ? cast_back(dh0, h0_type) : dh0};
  }
};

std::pair<Tensor, Tensor> diag_scan(const Tensor& x, const Tensor& g_in, const OptTensor& h0_, bool complement) {
  return guarded([&] {
    const Tensor h0_in = opt(h0_);
    need_cuda(x);
    need_device(x, g_in, h0_in);
    need_type(x, "x");
    need_float(g_in, "g");
    need_float(h0_in, "h0");
    need_shape(x.dim() >= 3 && g_in.sizes() == x.sizes(), "x, g [B, L, ...]");
    std::vector<int64_t> state_shape(x.sizes().begin(), x.sizes().end());
    state_shape.erase(state_shape.begin() + 1);
    if (h0_in.defined()) need_shape(h0_in.sizes() == at::IntArrayRef(state_shape), "h0 [B, ...] as x without its second dimension");
    refuse_tangents({x, g_in, h0_in});
    c10::cuda::CUDAGuard guard(x.device());
    const bool need = wants_grad({x, g_in, h0_in}), empty = x.numel() == 0;
    const auto o32 = x.options().dtype(at::kFloat);
    Tensor h, hT, states, g, xt;
    {
      at::NoGradGuard no_grad;
      g = in_type(g_in, x.scalar_type());
      const Tensor h0 = as32(h0_in);
      h = at::empty(x.sizes(), x.options());
      if (empty) {
        hT = h0.defined() ? h0.clone() : at::zeros(state_shape, o32);
      } else {
        xt = tokens(x);
        g = tokens(g);
        hT = at::empty(state_shape, o32);
        LetheGdnDiagArgs a = diag_args(xt, g, complement);
        a.h0 = ptr<float>(h0);
        a.h = ptr(h);
        a.hT = ptr<float>(hT);
        if (need) {
          states = at::empty({static_cast<int64_t>(lethe_gdn_diag_states_bytes(a.B, a.L, a.D, a.x_type) / 4)}, o32);
          a.states = ptr<float>(states);
        }
        const Tensor work = diag_work(&a, x, false);
        check(lethe_gdn_diag_forward(&a, stream_of(x)));
      }
    }
    if (need) {
      std::shared_ptr<DiagScanBackward> node(new DiagScanBackward(), torch::autograd::deleteNode);
      node->complement = complement;
      node->empty = empty;
      node->g_type = g_in.scalar_type();
      node->h0_type = h0_in.defined() ? h0_in.scalar_type() : at::kFloat;
      node->state_shape = state_shape;
      node->set_next_edges(torch::autograd::collect_next_edges(x, g_in, h0_in));
      node->keep(empty ? x : xt);
      node->keep(g);
      node->keep(states);
      torch::autograd::set_history(h, node);
      torch::autograd::set_history(hT, node);
    }
    return std::make_pair(h, hT);
  });
}

// whether some of t's memory may be some of the contiguous tensor `whole`'s: by addresses, since two storages can stand for the same memory
bool touches(const Tensor& t, const Tensor& whole) {
  if (t.numel() == 0 || lazy(t)) return false;      // (lazy: written out elsewhere)
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  const char *a = static_cast<const char*>(t.data_ptr()), *b = static_cast<const char*>(whole.data_ptr());
  return a < b + whole.nbytes() && b < a + (last + 1) * t.element_size();
}

Tensor diag_scan_step(const Tensor& x, const Tensor& g_in, const Tensor& state, bool complement) {
  return guarded([&] {
    need_cuda(state);
    if (state.scalar_type() != at::kFloat || !state.is_contiguous() || lazy(state) || state.dim() < 2)
      fail("the state must be a contiguous fp32 tensor [B, ...] (it is updated in place)");
    if (state.requires_grad()) fail("the state is updated in place and cannot require a gradient");
    need_device(state, x, g_in);
    need_type(x, "x");
    need_float(g_in, "g");
    need_shape(x.sizes() == state.sizes() && g_in.sizes() == state.sizes(), "x, g and state [B, ...]");
    refuse_tangents({x, g_in, state});
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(state.device());
    // what lies in the state's memory is read before any of it is written
    const auto readable = [&](const Tensor& t) {
      if (touches(t, state)) return t.clone(at::MemoryFormat::Contiguous);
      return lazy(t) || !packed_from(t, 1) ? as(t, t.scalar_type()) : t;
    };
    Tensor h = at::empty(x.sizes(), x.options());
    if (x.numel() == 0) return h;
    const Tensor xt = readable(x), g = readable(in_type(g_in, x.scalar_type()));
    LetheGdnDiagArgs a;
    memset(&a, 0, sizeof(a));
    a.B = state.size(0); a.L = 1; a.D = state.numel() / a.B;
    a.x_type = code(x.scalar_type()); a.g_type = code(g.scalar_type()); a.complement = complement;
    a.x = ptr(xt); a.x_batch = step_of(xt, 0);
    a.g = ptr(g); a.g_batch = step_of(g, 0);
    a.h = ptr(h);
    check(lethe_gdn_diag_step(&a, ptr<float>(state), stream_of(state)));
    if (!state.is_inference()) torch::autograd::impl::bump_version(state);
    return h;
  });
}

// ---------------------------------------------------------------------------------------------
// Norms around a block
// ---------------------------------------------------------------------------------------------
constexpr int64_t kMaxRow = 8192;

void check_row(const Tensor& x, double eps) {
  need_shape(x.dim() >= 1, "rows [..., D]");
  if (x.size(-1) < 1 || x.size(-1) > kMaxRow)
    fail("unsupported row length " + std::to_string(x.size(-1)) + " (need 1 to " + std::to_string(kMaxRow) + ")");
  if (!(eps >= 0.) || !std::isfinite(static_cast<float>(eps))) fail("eps must be a finite number in fp32, zero or more");
}
void check_vector(const Tensor& v, const Tensor& x, const char* name) {
  if (!v.defined()) return;
  need_float(v, name);
  if (v.dim() != 1 || v.size(0) != x.size(-1)) fail(std::string(name) + " must be a vector as long as a row");
}
// rows r = (i, j) of a tensor at i * outer + j * inner_stride, j over its dimension in front of the last
struct Rows {
  Tensor t;
  int64_t inner = 1, outer_stride = 0, inner_stride = 0;
};
Rows rows_of(const Tensor& t) {
  Rows r;
  r.t = lazy(t) || !packed_from(t, t.dim() - 1) || joint_stride(t, 0, t.dim() - 2) < 0 ? as(t, t.scalar_type()) : t;
  if (t.dim() >= 2) {
    r.inner = t.size(-2);
    r.inner_stride = t.size(-2) > 1 ? r.t.stride(-2) : 0;
    r.outer_stride = joint_stride(r.t, 0, t.dim() - 2);
  }
  return r;
}
// rows with one stride
Tensor even_rows(const Tensor& t, int64_t* stride) {
  const Tensor r = lazy(t) || !packed_from(t, t.dim() - 1) || joint_stride(t, 0, t.dim() - 1) < 0 ? as(t, t.scalar_type()) : t;
  *stride = joint_stride(r, 0, r.dim() - 1);
  return r;
}
Tensor norm_work(int64_t rows, int64_t D, int vectors, const Tensor& like, void** p, size_t* bytes) {
  Tensor w;
  if (!vectors) return w;
  *bytes = lethe_gdn_norm_work_bytes(rows, static_cast<int32_t>(D), vectors);
  w = at::empty({static_cast<int64_t>(*bytes)}, like.options().dtype(at::kByte));
  *p = ptr(w);
  return w;
}

LetheGdnGatedNormArgs gated_args(const Rows& x, const Rows& z, const Tensor& w, double eps, bool silu) {
  LetheGdnGatedNormArgs a;
  memset(&a, 0, sizeof(a));
  a.D = static_cast<int32_t>(x.t.size(-1));
  a.rows = x.t.numel() / a.D; a.inner = x.inner;
  a.x_type = code(x.t.scalar_type()); a.w_type = code(w.scalar_type()); a.silu = silu;
  a.eps = static_cast<float>(eps);
  a.x = ptr(x.t); a.x_outer = x.outer_stride; a.x_inner = x.inner_stride;
  a.gate = ptr(z.t); a.gate_outer = z.outer_stride; a.gate_inner = z.inner_stride;
  a.weight = ptr(w);
  return a;
}

struct GatedNormBackward : public FirstOrderNode {      // kept: x, gate, weight
  double eps = 0;
  bool silu = true;
  at::ScalarType w_type;
  std::string name() const override { return "GatedNormBackward"; }

  variable_list first_order(const variable_list& grads) override {
    auto self = getptr();
    const Tensor x = kept[0].unpack(self), z = kept[1].unpack(self), w = kept[2].unpack(self).contiguous();
    c10::cuda::CUDAGuard guard(x.device());
    Tensor dx, dz, dw;
    if (x.numel() == 0) {
      if (task_should_compute_output(2)) dw = at::zeros(w.sizes(), w.options().dtype(w_type));
      return {at::zeros(x.sizes(), x.options()), at::zeros(z.sizes(), z.options()), dw};
    }
    const Tensor dy = as(grads[0], x.scalar_type());
    const Rows xr = rows_of(x), zr = rows_of(z);
    LetheGdnGatedNormArgs a = gated_args(xr, zr, w, eps, silu);
    a.dy = ptr(dy);
    if (task_should_compute_output(0)) dx = at::empty(x.sizes(), x.options());
    if (task_should_compute_output(1)) dz = at::empty(z.sizes(), z.options());
    if (task_should_compute_output(2)) dw = at::empty(w.sizes(), w.options());
    a.dx = ptr(dx); a.dgate = ptr(dz); a.dweight = ptr(dw);
    const Tensor work = norm_work(a.rows, a.D, dw.defined(), x, &a.work, &a.work_bytes);
    check(lethe_gdn_gated_norm_vjp(&a, stream_of(x)));
    return {dx, dz, dw.defined() ? cast_back(dw, w_type) : dw};
  }
};

Tensor gated_norm(const Tensor& x, const Tensor& gate, const Tensor& weight, double eps, bool silu) {
  return guarded([&] {
    need_cuda(x);
    need_device(x, gate, weight);
    need_type(x, "x");
    check_row(x, eps);
    need_shape(gate.sizes() == x.sizes(), "x, gate [..., D]");
    if (gate.scalar_type() != x.scalar_type()) fail("the gate must have the type of x");
    check_vector(weight, x, "weight");
    refuse_tangents({x, gate, weight});
    c10::cuda::CUDAGuard guard(x.device());
    const bool need = wants_grad({x, gate, weight});
    Tensor y, w;
    Rows xr, zr;
    {
      at::NoGradGuard no_grad;
      w = in_type(weight, x.scalar_type());
      w = as(w, w.scalar_type());
      y = at::empty(x.sizes(), x.options());
      xr = rows_of(x);
      zr = rows_of(gate);
      if (x.numel()) {
        LetheGdnGatedNormArgs a = gated_args(xr, zr, w, eps, silu);
        a.y = ptr(y);
        check(lethe_gdn_gated_norm(&a, stream_of(x)));
      }
    }
    if (need) {
      std::shared_ptr<GatedNormBackward> node(new GatedNormBackward(), torch::autograd::deleteNode);
      node->eps = eps;
      node->silu = silu;
      node->w_type = weight.scalar_type();
      node->set_next_edges(torch::autograd::collect_next_edges(x, gate, weight));
      node->keep(xr.t);
      node->keep(zr.t);
      node->keep(w);
      torch::autograd::set_history(y, node);
    }
    return y;
  });
}

struct Vectors {
  Tensor w, pw, scale;      // one type, contiguous
};

LetheGdnResidualNormArgs residual_args(const Tensor& r, at::ScalarType x_type, const Vectors& v, double eps, double scale_value) {
  LetheGdnResidualNormArgs a;
  memset(&a, 0, sizeof(a));
  a.D = static_cast<int32_t>(r.size(-1));
  a.rows = r.numel() / a.D;
  a.x_type = code(x_type); a.r_type = code(r.scalar_type()); a.w_type = code(v.w.scalar_type());
  a.eps = static_cast<float>(eps); a.scale_value = static_cast<float>(scale_value);
  a.weight = ptr(v.w); a.post_weight = ptr(v.pw); a.scale = ptr(v.scale);
  a.r = ptr(r);
  return a;
}

struct ResidualNormBackward : public FirstOrderNode {      // kept: r, x (where needed), weight, post_weight, scale
  double eps = 0, scale_value = 1;
  at::ScalarType x_type, types[3];      // of weight, post_weight, scale as they came
  bool has_residual = true;
  std::string name() const override { return "ResidualNormBackward"; }

  variable_list first_order(const variable_list& grads) override {
    auto self = getptr();
    const Tensor r_kept = kept[0].unpack(self), x = kept[1].unpack(self);
    const auto vec = [&](int i) { const Tensor t = kept[i].unpack(self); return t.defined() ? t.contiguous() : t; };
    const Vectors v{vec(2), vec(3), vec(4)};
    const Tensor r = r_kept.contiguous();
    c10::cuda::CUDAGuard guard(r.device());
    const auto xo = r.options().dtype(x_type);
    const bool want_x = task_should_compute_output(0), want_res = has_residual && task_should_compute_output(1);
    const Tensor* given[3] = {&v.w, &v.pw, &v.scale};
    Tensor dx, dres, dv[3];
    const auto result = [&]() -> variable_list {
      variable_list out(5);
      if (want_x) out[0] = dx;
      if (want_res) out[1] = dres;
      for (int i = 0; i < 3; ++i)
        if (dv[i].defined()) out[2 + i] = cast_back(dv[i], types[i]);
      return out;
    };
    const bool none = r.numel() == 0;
    for (int i = 0; i < 3; ++i)
      if (given[i]->defined() && task_should_compute_output(2 + i)) dv[i] = none ? at::zeros_like(*given[i]) : at::empty_like(*given[i]);
    if (none) {
      dx = at::zeros(r.sizes(), xo);
      dres = at::zeros(r.sizes(), r.options());
      return result();
    }
    const Tensor dy = grads[0].defined() ? as(grads[0], x_type) : Tensor(), dr = grads[1].defined() ? as(grads[1], r.scalar_type()) : Tensor();
    LetheGdnResidualNormArgs a = residual_args(r, x_type, v, eps, scale_value);
    Tensor xr;
    if (x.defined()) {
      xr = even_rows(x, &a.x_stride);
      a.x = ptr(xr);
    }
    a.dy = ptr(dy); a.dr = ptr(dr);
    // nothing between the sum and x: one gradient for both
    const bool same = !v.pw.defined() && !v.scale.defined() && scale_value == 1. && x_type == r.scalar_type();
    if (want_res || (same && want_x)) dres = at::empty(r.sizes(), r.options());
    if (want_x) dx = same ? dres : at::empty(r.sizes(), xo);
    a.dresidual = ptr(dres);
    if (!same) a.dx = ptr(dx);
    a.dweight = ptr(dv[0]); a.dpost_weight = ptr(dv[1]); a.dscale = ptr(dv[2]);
    const int n = dv[0].defined() + dv[1].defined() + dv[2].defined();
    const Tensor work = norm_work(a.rows, a.D, n, r, &a.work, &a.work_bytes);
    check(lethe_gdn_residual_norm_vjp(&a, stream_of(r)));
    return result();
  }
};

std::pair<Tensor, Tensor> residual_norm(const Tensor& x, const OptTensor& residual_, const Tensor& weight, const OptTensor& post_,
                                        const OptTensor& scale_, double eps, double scale_value) {
  return guarded([&] {
    const Tensor residual = opt(residual_), post = opt(post_), scale = opt(scale_);
    need_cuda(x);
    need_device(x, residual, weight, post, scale);
    need_type(x, "x");
    check_row(x, eps);
    if (std::isfinite(scale_value) && !std::isfinite(static_cast<float>(scale_value))) fail("scale lies beyond what fp32 holds");
    if (residual.defined()) {
      need_shape(residual.sizes() == x.sizes(), "x, residual [..., D]");
      if (residual.scalar_type() != at::kFloat && residual.scalar_type() != x.scalar_type())
        fail("the residual stream must be fp32 or have the type of x");
    }
    check_vector(weight, x, "weight");
    check_vector(post, x, "post_weight");
    check_vector(scale, x, "scale");
    refuse_tangents({x, residual, weight, post, scale});
    c10::cuda::CUDAGuard guard(x.device());
    const bool need = wants_grad({x, residual, weight, post, scale});
    Vectors v;
    Tensor xr, r, y;
    {
      at::NoGradGuard no_grad;
      // one type for the vectors: that of all of them, if it is fp32 or that of x, else fp32
      const auto dt = weight.scalar_type();
      bool one = dt == at::kFloat || dt == x.scalar_type();
      for (const Tensor* t : {&post, &scale}) one = one && (!t->defined() || t->scalar_type() == dt);
      const auto vec = [&](const Tensor& t) { return t.defined() ? as(t, one ? dt : at::kFloat) : t; };
      v = {vec(weight), vec(post), vec(scale)};
      y = at::empty(x.sizes(), x.options());
      r = at::empty(x.sizes(), residual.defined() ? residual.options() : x.options());
      int64_t x_stride = 0, res_stride = 0;
      xr = even_rows(x, &x_stride);
      if (x.numel()) {
        LetheGdnResidualNormArgs a = residual_args(r, x.scalar_type(), v, eps, scale_value);
        Tensor res;
        if (residual.defined()) {
          res = even_rows(residual, &res_stride);
          a.residual = ptr(res);
          a.residual_stride = res_stride;
        }
        a.x = ptr(xr);
        a.x_stride = x_stride;
        a.y = ptr(y);
        check(lethe_gdn_residual_norm(&a, stream_of(x)));
      }
    }
    if (need) {
      std::shared_ptr<ResidualNormBackward> node(new ResidualNormBackward(), torch::autograd::deleteNode);
      node->eps = eps;
      node->scale_value = scale_value;
      node->x_type = x.scalar_type();
      node->has_residual = residual.defined();
      node->types[0] = weight.scalar_type();
      node->types[1] = post.defined() ? post.scalar_type() : at::kFloat;
      node->types[2] = scale.defined() ? scale.scalar_type() : at::kFloat;
      node->set_next_edges(torch::autograd::collect_next_edges(x, residual, weight, post, scale));
      torch::autograd::set_history(y, node);
      torch::autograd::set_history(r, node);
      node->keep(r, true);
      const bool need_x = post.defined() || (scale.defined() && scale.requires_grad());
      node->keep(need_x ? xr : Tensor());
      node->keep(v.w);
      node->keep(v.pw);
      node->keep(v.scale);
    }
    return std::make_pair(y, r);
  });
}

}  // namespace

void bind_block(pybind11::module_& m) {
  m.def("diag_scan", &diag_scan);
  m.def("diag_scan_step", &diag_scan_step);
  m.def("gated_norm", &gated_norm);
  m.def("residual_norm", &residual_norm);
}

}  // namespace lethe_torch
