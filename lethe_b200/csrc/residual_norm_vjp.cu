// The vector-Jacobian product of the residual sum and the norm behind it: residual_norm.cuh.
#include "residual_norm.cuh"
#include "umma.cuh"

namespace lg {

template <int XT, int RT, typename S, int BRANCH>
using ResidualRingBack = RowRing<S, S::R * 8 * (elem_bytes(XT) * (BRANCH ? 2 : 1) + 2 * elem_bytes(RT)), residual_ctas<S>(true), std::min(elem_bytes(XT), elem_bytes(RT))>;


// BRANCH 0: nothing of x is needed.  1: x for dscale.  2: norm of x.  Both gradients of the branch come from one sum over rows: with
// q = sum of d n1, dscale = post_weight q and dpost_weight = scale q (without a norm of x: q = sum of d x = dscale).
template <int XT, int RT, typename S, int BRANCH>
__global__ void __launch_bounds__(S::kThreads, residual_ctas<S>(true)) residual_norm_vjp_kernel(const ResidualProblem p) {
  using Ring = ResidualRingBack<XT, RT, S, BRANCH>;
  constexpr int kR = 0, kDr = S::R * elem_bytes(RT) / 2, kDy = 2 * kDr, kX = kDy + S::R * elem_bytes(XT) / 2;
  __shared__ __align__(16) float sums[2][2][3][S::kWarps];
  extern __shared__ __align__(16) unsigned char smem[];
  const Ring ring(smem);
  const int t = threadIdx.x % S::T;
  const Turns turns(p.rows, S::kRows, threadIdx.x / S::T);
  RowPtr pr(p.r, turns, p.D, elem_bytes(RT)), pdr(p.dr, turns, p.D, elem_bytes(RT)), pdy(p.dy, turns, p.D, elem_bytes(XT)), px(p.x, turns, p.x_stride, elem_bytes(XT));
  RowPtr pdres(p.dres, turns, p.D, elem_bytes(RT)), pdx(p.dx, turns, p.D, elem_bytes(XT));
  const auto next = [&] {
    pr.next();
    pdr.next();
    pdy.next();
    if constexpr (BRANCH >= 1) px.next();
  };
  int far = 0;
  const auto fetch = [&](int stage) {
    if (far < turns.mine) {
      ring.template copy<RT, kR>(stage, pr.p, t, p.D);
      if (p.dr) ring.template copy<RT, kDr>(stage, pdr.p, t, p.D);
      if (p.dy) ring.template copy<XT, kDy>(stage, pdy.p, t, p.D);
      if constexpr (BRANCH >= 1) ring.template copy<XT, kX>(stage, px.p, t, p.D);
    }
    Ring::commit();
    ++far;
    next();
  };
  if constexpr (Ring::kOn)
    for (int i = 0; i < Ring::kStages - 1; ++i) fetch(i);
  F2 w[S::P], sc[S::P], acc_w[S::P], acc_q[S::P];      // sc: scale, times post_weight where there is one
  S::template vector<XT>(w, p.w, p.w_f32, t, p.D, 0.f);
  S::template vector<XT>(sc, p.scale, p.w_f32, t, p.D, p.scale_value);
  if constexpr (BRANCH == 2) {
    F2 pw[S::P];
    S::template vector<XT>(pw, p.pw, p.w_f32, t, p.D, 0.f);
#pragma unroll
    for (int n = 0; n < S::P; ++n) sc[n] = sc[n] * pw[n];
  }
#pragma unroll
  for (int n = 0; n < S::P; ++n) acc_w[n] = acc_q[n] = f2(0.f);
  const float over = 1.f / p.D;
  int flip = 0, stage = 0;
  for (int turn = 0; turn < turns.all; ++turn, flip ^= 1, pdres.next(), pdx.next()) {
    const bool live = turn < turns.mine;
    Raw<XT, 8> x[S::R], dy[S::R];
    Raw<RT, 8> r[S::R], dr[S::R];
    if constexpr (Ring::kOn) {
      Ring::wait();
      ring.template take<RT, kR>(r, stage);
      ring.template take<RT, kDr>(dr, stage);
      ring.template take<XT, kDy>(dy, stage);
      if constexpr (BRANCH >= 1) ring.template take<XT, kX>(x, stage);
      fetch(stage ? stage - 1 : Ring::kStages - 1);
      stage = stage + 1 == Ring::kStages ? 0 : stage + 1;
    }
    if (!Ring::kOn || !live) {      // (a row that is not there adds nothing)
#pragma unroll
      for (int i = 0; i < S::R; ++i) {
        x[i].zero();
        dy[i].zero();
        r[i].zero();
        dr[i].zero();
      }
    }
    if constexpr (!Ring::kOn) {
      if (live) {
        S::template load<RT>(r, pr.p, t, p.D);
        if (p.dy) S::template load<XT>(dy, pdy.p, t, p.D);
        if (p.dr) S::template load<RT>(dr, pdr.p, t, p.D);
        if constexpr (BRANCH >= 1) S::template load<XT>(x, px.p, t, p.D);
      }
      next();
    }
    constexpr int K = BRANCH == 2 ? 3 : 2;
    F2 sum[3] = {f2(0.f), f2(0.f), f2(0.f)};
#pragma unroll
    for (int n = 0; n < S::P; ++n) {
      const F2 rv = r[n / 4].get2(n % 4);
      sum[0] = fma2(rv, rv, sum[0]);
      sum[1] = fma2(dy[n / 4].get2(n % 4) * w[n], rv, sum[1]);
      if constexpr (BRANCH == 2) sum[2] = fma2(x[n / 4].get2(n % 4), x[n / 4].get2(n % 4), sum[2]);
    }
    float s[K];
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = lo(sum[k]) + hi(sum[k]);
    S::template row_sums<K>(s, sums[flip][0]);
    const float root = live ? rsqrtf(fmaf(s[0], over, p.eps)) : 0.f;      // (with eps = 0 a row that is not there would have an infinite root)
    const F2 r2 = f2(root), c2 = f2(-s[1] * over * root * root);
    F2 r1 = f2(1.f);
    if constexpr (BRANCH == 2) r1 = f2(live ? rsqrtf(fmaf(s[2], over, p.eps)) : 0.f);
    F2 d[S::P], qq = f2(0.f);
#pragma unroll
    for (int n = 0; n < S::P; ++n) {
      const F2 rv = r[n / 4].get2(n % 4), dyv = dy[n / 4].get2(n % 4);
      acc_w[n] = fma2(dyv, rv * r2, acc_w[n]);
      d[n] = fma2(r2, fma2(rv, c2, dyv * w[n]), dr[n / 4].get2(n % 4));
      if constexpr (BRANCH == 1) acc_q[n] = fma2(d[n], x[n / 4].get2(n % 4), acc_q[n]);
      if constexpr (BRANCH == 2) {
        const F2 dn = d[n] * (x[n / 4].get2(n % 4) * r1);
        acc_q[n] = acc_q[n] + dn;
        qq = fma2(dn, sc[n], qq);
      }
    }
    if (live && p.dres) S::template store<RT>(d, pdres.p, t, p.D);
    if constexpr (BRANCH == 2) {
      float q[1] = {lo(qq) + hi(qq)};
      S::template row_sums<1>(q, sums[flip][1]);
      const F2 c1 = f2(-q[0] * over) * r1;
#pragma unroll
      for (int n = 0; n < S::P; ++n) d[n] = r1 * fma2(x[n / 4].get2(n % 4), c1, d[n] * sc[n]);
    } else {
#pragma unroll
      for (int n = 0; n < S::P; ++n) d[n] = d[n] * sc[n];
    }
    if (live && p.dx) S::template store<XT>(d, pdx.p, t, p.D);
  }
  if (!p.part) return;
  griddep_launch();      // (the kernel that adds the shares waits for their stores)
  float* line = p.part + static_cast<long long>(blockIdx.x) * p.vectors * p.D;
  float* columns = reinterpret_cast<float*>(smem);
  if (p.at[0] >= 0) S::column_share(acc_w, line + static_cast<long long>(p.at[0]) * p.D, columns, t, p.D);
  if constexpr (BRANCH == 2) {
    F2 v[S::P];
    S::template vector<XT>(v, p.scale, p.w_f32, t, p.D, p.scale_value);
#pragma unroll
    for (int n = 0; n < S::P; ++n) v[n] = v[n] * acc_q[n];
    if (p.at[1] >= 0) S::column_share(v, line + static_cast<long long>(p.at[1]) * p.D, columns, t, p.D);
    S::template vector<XT>(v, p.pw, p.w_f32, t, p.D, 0.f);
#pragma unroll
    for (int n = 0; n < S::P; ++n) acc_q[n] = acc_q[n] * v[n];
  }
  if constexpr (BRANCH >= 1)
    if (p.at[2] >= 0) S::column_share(acc_q, line + static_cast<long long>(p.at[2]) * p.D, columns, t, p.D);
}

}  // namespace lg

extern "C" int lethe_gdn_residual_norm_vjp(const LetheGdnResidualNormArgs* a, void* stream) {
  using namespace lg;
  ResidualProblem p;
  if (int e = residual_problem(a, &p, true)) return e;
  if (a->dpost_weight && !a->post_weight) return kErrFlags;
  ColumnSums c{};
  void* const wanted[3] = {a->dweight, a->dpost_weight, a->dscale};
  for (int i = 0; i < 3; ++i)
    if (wanted[i]) {
      p.at[i] = p.vectors;
      c.out[p.vectors] = wanted[i];
      c.f32[p.vectors++] = p.w_f32;
    }
  if (p.vectors) {
    if (!a->work) return kErrNull;
    if (a->work_bytes < lethe_gdn_norm_work_bytes(a->rows, a->D, p.vectors)) return kErrWorkspace;
    if (reinterpret_cast<uintptr_t>(a->work) & 15) return kErrAlign;
    p.part = static_cast<float*>(a->work);
  }
  DeviceGuard guard(a->r);
  if (!guard.ok) return kErrDevice;
  const int branch = p.pw ? 2 : a->dscale ? 1 : 0;
  const int w = widest_piece(widest_of(a->x_type, a->r_type), p.D, [&](int n) {
    return (!branch || piece_aligned(n, p.x, a->x_type, p.x_stride)) && piece_aligned(n, p.r, a->r_type) && piece_aligned(n, p.dy, a->x_type) &&
           piece_aligned(n, p.dr, a->r_type) && piece_aligned(n, p.dx, a->x_type) && piece_aligned(n, p.dres, a->r_type);
  });
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int grid = 0;
  const auto run = [&](auto kind) {
    constexpr int kBranch = decltype(kind)::value;
    return by_stream_type(a->x_type, a->r_type, [&](auto x, auto r) {
      return by_row_shape<widest_of(x.value, r.value)>(p.D, w, [&](auto s) {
        using S = decltype(s);
        grid = std::min(norm_grid(p.rows, S::kRows, residual_ctas<S>(true)), norm_parts_max(p.D));
        const auto kern = residual_norm_vjp_kernel<x.value, r.value, S, kBranch>;
        constexpr int smem = std::max(ResidualRingBack<x.value, r.value, S, kBranch>::kBytes, S::kColumnBytes);
        static SmemAttr attr;
        if (int e = attr.set(kern, smem)) return e;
        kern<<<grid, S::kThreads, smem, st>>>(p);
        return launched_ok();
      });
    });
  };
  const int e = branch == 2   ? run(std::integral_constant<int, 2>())
                : branch == 1 ? run(std::integral_constant<int, 1>())
                              : run(std::integral_constant<int, 0>());
  if (e || !p.part) return e;
  c.part = p.part;
  c.parts = grid;
  c.vectors = p.vectors;
  c.D = p.D;
  c.x_type = a->x_type;
  return launch_column_sums(c, st);
}
