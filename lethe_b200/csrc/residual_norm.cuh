// The residual sum and the norm in front of the next block, and its vector-Jacobian product.
//
//   t = x, or n1 pw with n1 = x r1, r1 = rsqrt(mean x^2 + eps);   r = residual + scale t, rounded to the stream's type
//   y = n2 w, n2 = r r2, r2 = rsqrt(mean r^2 + eps)
//   d = dr + r2 (dy w - n2 mean(dy w n2)) = dresidual;   dweight = sum over rows of dy n2,  dscale = sum of d t
//   dx = scale d,  or r1 (u pw - n1 mean(u pw n1)) with u = scale d;  dpost_weight = sum of u n1
//
// Bound by HBM.  The backward takes n2 from r as it was stored, so it reads the stream once and x only where the branch has
// something to learn.  Measured (16384 x 4096 bf16, norms on both sides, learned scale): 92 us forward, 0.89 of the measured copy bandwidth,
// 151 backward, 0.81; without a branch to learn 96 and 92, 0.98 in all.
#pragma once
#include "block_norm.cuh"

namespace lg {

struct ResidualProblem {
  long long rows;
  int D, w_f32;
  float eps, scale_value;
  const void* x;
  long long x_stride;
  const void* res;
  long long res_stride;
  const void *w, *pw, *scale;
  void *r, *y;
  const void *dy, *dr;
  void *dx, *dres;
  float *part;              // per CTA: the vectors that are wanted, in the order dweight, dpost_weight, dscale
  int vectors, at[3];       // their number, and the place of each (-1: not wanted)
};

// CTAs on an SM: registers (64 a thread forward, 128 backward and with two pieces)
template <typename S> constexpr int residual_ctas(bool backward) { return (backward || S::R > 1 ? 512 : 1024) / S::kThreads; }
// f(XT, RT)
template <typename F>
int by_stream_type(int xt, int rt, F&& f) {
  using T32 = std::integral_constant<int, LETHE_F32>;
  if (rt == LETHE_F32) return by_x_type(xt, [&](auto x) { return f(x, T32()); });
  return by_x_type(xt, [&](auto x) { return f(x, x); });
}

inline int residual_problem(const LetheGdnResidualNormArgs* a, ResidualProblem* p, bool backward) {
  if (!a) return kErrNull;
  if (a->rows <= 0 || a->D <= 0 || a->D > kNormMaxD || !norm_types_ok(a->x_type, a->w_type) || !norm_types_ok(a->x_type, a->r_type) || !(a->eps >= 0.f) || !std::isfinite(a->eps))
    return kErrDims;
  if (!a->r || !a->weight || (!backward && (!a->x || !a->y))) return kErrNull;
  if (backward && !a->x && (a->post_weight || a->dscale)) return kErrNull;
  if (!on_elements(a->x_type, a->x, a->y, a->dy, a->dx) || !on_elements(a->r_type, a->residual, a->r, a->dr, a->dresidual) ||
      !on_elements(a->w_type, a->weight, a->post_weight, a->scale, a->dweight, a->dpost_weight, a->dscale)) return kErrAlign;
  *p = {a->rows, a->D, a->w_type == LETHE_F32, a->eps, a->scale_value, a->x, a->x_stride, a->residual, a->residual_stride, a->weight, a->post_weight,
        a->scale, a->r, a->y, a->dy, a->dr, a->dx, a->dresidual, nullptr, 0, {-1, -1, -1}};
  return kOk;
}

}  // namespace lg
