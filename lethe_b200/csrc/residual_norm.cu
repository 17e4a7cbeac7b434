// The residual sum and the norm in front of the next block: residual_norm.cuh.
#include "residual_norm.cuh"

namespace lg {

template <int XT, int RT, typename S> using ResidualRing = RowRing<S, S::R * 8 * (elem_bytes(XT) + elem_bytes(RT)), residual_ctas<S>(false), std::min(elem_bytes(XT), elem_bytes(RT))>;

template <int XT, int RT, typename S, bool POST>
__global__ void __launch_bounds__(S::kThreads, residual_ctas<S>(false)) residual_norm_kernel(const ResidualProblem p) {
  using Ring = ResidualRing<XT, RT, S>;
  constexpr int kX = 0, kRes = S::R * elem_bytes(XT) / 2;
  __shared__ __align__(16) float sums[2][2][1][S::kWarps];
  extern __shared__ __align__(16) unsigned char smem[];
  const Ring ring(smem);
  const int t = threadIdx.x % S::T;
  const Turns turns(p.rows, S::kRows, threadIdx.x / S::T);
  RowPtr px(p.x, turns, p.x_stride, elem_bytes(XT)), pres(p.res, turns, p.res_stride, elem_bytes(RT));      // of the copies, or of the rows themselves
  RowPtr pr(p.r, turns, p.D, elem_bytes(RT)), py(p.y, turns, p.D, elem_bytes(XT));
  int far = 0;
  const auto fetch = [&](int stage) {
    if (far < turns.mine) {
      ring.template copy<XT, kX>(stage, px.p, t, p.D);
      if (p.res) ring.template copy<RT, kRes>(stage, pres.p, t, p.D);      // (else the cells stay zeros)
    }
    Ring::commit();
    ++far;
    px.next();
    pres.next();
  };
  if constexpr (Ring::kOn)
    for (int i = 0; i < Ring::kStages - 1; ++i) fetch(i);
  F2 w[S::P], sc[S::P], pw[S::P];
  S::template vector<XT>(w, p.w, p.w_f32, t, p.D, 0.f);
  S::template vector<XT>(sc, p.scale, p.w_f32, t, p.D, p.scale_value);
  if constexpr (POST) S::template vector<XT>(pw, p.pw, p.w_f32, t, p.D, 0.f);
  const float over = 1.f / p.D;
  int flip = 0, stage = 0;
  for (int turn = 0; turn < turns.all; ++turn, flip ^= 1, pr.next(), py.next()) {
    const bool live = turn < turns.mine;
    Raw<XT, 8> x[S::R];
    Raw<RT, 8> res[S::R];
    if constexpr (Ring::kOn) {
      Ring::wait();
      ring.template take<XT, kX>(x, stage);
      ring.template take<RT, kRes>(res, stage);
      fetch(stage ? stage - 1 : Ring::kStages - 1);
      stage = stage + 1 == Ring::kStages ? 0 : stage + 1;
    } else {
#pragma unroll
      for (int i = 0; i < S::R; ++i) {
        x[i].zero();
        res[i].zero();
      }
      if (live) {
        S::template load<XT>(x, px.p, t, p.D);
        if (p.res) S::template load<RT>(res, pres.p, t, p.D);
      }
      px.next();
      pres.next();
    }
    F2 r1 = f2(1.f);
    if constexpr (POST) {
      F2 xx = f2(0.f);
#pragma unroll
      for (int n = 0; n < S::P; ++n) xx = fma2(x[n / 4].get2(n % 4), x[n / 4].get2(n % 4), xx);
      float s[1] = {lo(xx) + hi(xx)};
      S::template row_sums<1>(s, sums[flip][0]);
      r1 = f2(rsqrtf(fmaf(s[0], over, p.eps)));
    }
    Raw<RT, 8> kept[S::R];
    F2 rr = f2(0.f);
#pragma unroll
    for (int n = 0; n < S::P; ++n) {
      F2 b = x[n / 4].get2(n % 4);
      if constexpr (POST) b = b * r1 * pw[n];
      // product and sum are rounded each, as the formula reads: with one rounding a sum could fall to the other side of a tie of the stored type
      kept[n / 4].set2(n % 4, res[n / 4].get2(n % 4) + b * sc[n]);
      const F2 v = kept[n / 4].get2(n % 4);
      rr = fma2(v, v, rr);
    }
    if (live) S::template store<RT>(kept, pr.p, t, p.D);
    float s[1] = {lo(rr) + hi(rr)};
    S::template row_sums<1>(s, sums[flip][1]);
    const F2 r2 = f2(rsqrtf(fmaf(s[0], over, p.eps)));
    F2 y[S::P];
#pragma unroll
    for (int n = 0; n < S::P; ++n) y[n] = kept[n / 4].get2(n % 4) * r2 * w[n];
    if (live) S::template store<XT>(y, py.p, t, p.D);
  }
}

}  // namespace lg

extern "C" int lethe_gdn_residual_norm(const LetheGdnResidualNormArgs* a, void* stream) {
  using namespace lg;
  ResidualProblem p;
  if (int e = residual_problem(a, &p, false)) return e;
  DeviceGuard guard(a->r);
  if (!guard.ok) return kErrDevice;
  const int w = widest_piece(widest_of(a->x_type, a->r_type), p.D, [&](int n) {
    return piece_aligned(n, p.x, a->x_type, p.x_stride) && piece_aligned(n, p.res, a->r_type, p.res_stride) && piece_aligned(n, p.r, a->r_type) &&
           piece_aligned(n, p.y, a->x_type);
  });
  return by_stream_type(a->x_type, a->r_type, [&](auto x, auto r) {
    return by_row_shape<widest_of(x.value, r.value)>(p.D, w, [&](auto s) {
      using S = decltype(s);
      const int grid = norm_grid(p.rows, S::kRows, residual_ctas<S>(false));
      constexpr int smem = ResidualRing<x.value, r.value, S>::kBytes;
      cudaStream_t st = static_cast<cudaStream_t>(stream);
      const auto go = [&](auto kern, SmemAttr& attr) {
        if (int e = attr.set(kern, smem)) return e;
        kern<<<grid, S::kThreads, smem, st>>>(p);
        return launched_ok();
      };
      static SmemAttr attr[2];
      return p.pw ? go(residual_norm_kernel<x.value, r.value, S, true>, attr[1]) : go(residual_norm_kernel<x.value, r.value, S, false>, attr[0]);
    });
  });
}
