// The norm behind a block, y = x / rms(x) * weight * act(gate), its vector-Jacobian product, and the column sums of both norms.
//
//   r = rsqrt(mean x^2 + eps), n = x r, a = act(gate) (logistic s, or gate s), y = n w a
//   dgate = dy n w a',  a' = s (1 - s) or s (1 + gate (1 - s));   dweight = sum over rows of dy n a
//   dn = dy w a,  dx = r (dn - n mean(dn n))
//
// Bound by HBM: 6 bytes a value forward and 10 backward in 16 bits.  mean(dn n) = r mean(dn x), so both row sums of the backward
// are of what was loaded and are formed together.  Measured (4 x 4096 x 16 rows of 128 bf16): 38 us forward, 0.81 of the measured copy
// bandwidth, 68 backward, 0.75 with the column sums; each alone on a cold cache 31 and 56 us.
#include "block_norm.cuh"
#include "umma.cuh"

namespace lg {

struct GatedProblem {
  long long rows, inner;
  int D, w_f32;
  float eps;
  const void* x;
  long long xo, xi;
  const void* z;
  long long zo, zi;
  const void* w;
  void* y;
  const void* dy;
  void *dx, *dz;
  float* part;      // per CTA the sums for dweight; NULL: not wanted
};

// logistic function s = 1 / (1 + e), e = exp(-z).  Results in 32 bits: the exponential is expf, the quotient good to 2 ulp up to a divisor of
// 2^126 and 0 beyond, that is for gates below -87.3.  In 16 bits: exponential and reciprocal by the approximations, 2^-22 off each, and with the
// rounding of its argument the exponential is off by |z| 2^-24 of itself more.
template <int XT>
__device__ __forceinline__ F2 logistic(F2 z, F2& e) {
  float a, b;
  if constexpr (XT == LETHE_F32) {
    a = expf(-lo(z));
    b = expf(-hi(z));
    e = f2(a, b);
    return f2(__fdividef(1.f, 1.f + a), __fdividef(1.f, 1.f + b));
  }
  const F2 t = z * f2(-1.4426950408889634f);
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(lo(t)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(hi(t)));
  e = f2(a, b);
  const F2 d = e + f2(1.f);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(a) : "f"(lo(d)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(b) : "f"(hi(d)));
  return f2(a, b);
}
// 1 - s = e s: by subtraction a gate of 12 would leave percents of it.  (Where e is infinite, s is 0.)
__device__ __forceinline__ F2 one_less(F2 s, F2 e) { return f2(fminf(lo(e), 3e38f), fminf(hi(e), 3e38f)) * s; }

// CTAs on an SM: registers (64 a thread forward, 80 backward; twice that with two pieces)
template <typename S> constexpr int gated_ctas(bool backward) { return S::R > 1 ? 512 / S::kThreads : (backward ? 768 : 1024) / S::kThreads; }
template <int XT, typename S, bool BACK> using GatedRing = RowRing<S, (BACK ? 3 : 2) * S::R * 8 * elem_bytes(XT), gated_ctas<S>(BACK), elem_bytes(XT)>;

template <int XT, bool SILU, typename S>
__global__ void __launch_bounds__(S::kThreads, gated_ctas<S>(false)) gated_norm_kernel(const GatedProblem p) {
  using Ring = GatedRing<XT, S, false>;
  constexpr int kX = 0, kZ = S::R * elem_bytes(XT) / 2;
  __shared__ __align__(16) float sums[2][1][S::kWarps];
  extern __shared__ __align__(16) unsigned char smem[];
  const Ring ring(smem);
  const int t = threadIdx.x % S::T;
  const Turns turns(p.rows, S::kRows, threadIdx.x / S::T);
  RowWalk walk(turns, p.inner);
  WalkPtr px(p.x, walk, p.xo, p.xi, elem_bytes(XT)), pz(p.z, walk, p.zo, p.zi, elem_bytes(XT));      // of the copies, or of the rows themselves
  RowPtr py(p.y, turns, p.D, elem_bytes(XT));
  const auto next = [&] {
    const bool round = walk.next();
    px.next(round);
    pz.next(round);
  };
  int far = 0;
  const auto fetch = [&](int stage) {
    if (far < turns.mine) {
      ring.template copy<XT, kX>(stage, px.p, t, p.D);
      ring.template copy<XT, kZ>(stage, pz.p, t, p.D);
    }
    Ring::commit();
    ++far;
    next();
  };
  if constexpr (Ring::kOn)
    for (int i = 0; i < Ring::kStages - 1; ++i) fetch(i);
  F2 w[S::P];
  S::template vector<XT>(w, p.w, p.w_f32, t, p.D, 0.f);
  const float over = 1.f / p.D;
  int flip = 0, stage = 0;
  for (int turn = 0; turn < turns.all; ++turn, flip ^= 1, py.next()) {
    const bool live = turn < turns.mine;
    Raw<XT, 8> x[S::R], z[S::R];
    if constexpr (Ring::kOn) {
      Ring::wait();
      ring.template take<XT, kX>(x, stage);
      ring.template take<XT, kZ>(z, stage);
      fetch(stage ? stage - 1 : Ring::kStages - 1);
      stage = stage + 1 == Ring::kStages ? 0 : stage + 1;
    } else {
#pragma unroll
      for (int i = 0; i < S::R; ++i) {
        x[i].zero();
        z[i].zero();
      }
      if (live) {
        S::template load<XT>(x, px.p, t, p.D);
        S::template load<XT>(z, pz.p, t, p.D);
      }
      next();
    }
    F2 xx = f2(0.f);
#pragma unroll
    for (int n = 0; n < S::P; ++n) xx = fma2(x[n / 4].get2(n % 4), x[n / 4].get2(n % 4), xx);
    float s[1] = {lo(xx) + hi(xx)};
    S::template row_sums<1>(s, sums[flip]);
    const F2 r = f2(rsqrtf(fmaf(s[0], over, p.eps)));
    F2 y[S::P];
#pragma unroll
    for (int n = 0; n < S::P; ++n) {
      F2 e;
      const F2 zv = z[n / 4].get2(n % 4), sg = logistic<XT>(zv, e);
      y[n] = x[n / 4].get2(n % 4) * r * w[n] * (SILU ? zv * sg : sg);
    }
    if (live) S::template store<XT>(y, py.p, t, p.D);
  }
}

template <int XT, bool SILU, typename S>
__global__ void __launch_bounds__(S::kThreads, gated_ctas<S>(true)) gated_norm_vjp_kernel(const GatedProblem p) {
  using Ring = GatedRing<XT, S, true>;
  constexpr int kEach = S::R * elem_bytes(XT) / 2, kX = 0, kZ = kEach, kD = 2 * kEach;
  __shared__ __align__(16) float sums[2][2][S::kWarps];
  extern __shared__ __align__(16) unsigned char smem[];
  const Ring ring(smem);
  const int t = threadIdx.x % S::T;
  const Turns turns(p.rows, S::kRows, threadIdx.x / S::T);
  RowWalk walk(turns, p.inner);
  WalkPtr px(p.x, walk, p.xo, p.xi, elem_bytes(XT)), pz(p.z, walk, p.zo, p.zi, elem_bytes(XT));
  RowPtr pd(p.dy, turns, p.D, elem_bytes(XT)), pdx(p.dx, turns, p.D, elem_bytes(XT)), pdz(p.dz, turns, p.D, elem_bytes(XT));
  const auto next = [&] {
    const bool round = walk.next();
    px.next(round);
    pz.next(round);
    pd.next();
  };
  int far = 0;
  const auto fetch = [&](int stage) {
    if (far < turns.mine) {
      ring.template copy<XT, kX>(stage, px.p, t, p.D);
      ring.template copy<XT, kZ>(stage, pz.p, t, p.D);
      ring.template copy<XT, kD>(stage, pd.p, t, p.D);
    }
    Ring::commit();
    ++far;
    next();
  };
  if constexpr (Ring::kOn)
    for (int i = 0; i < Ring::kStages - 1; ++i) fetch(i);
  F2 w[S::P], acc[S::P];
  S::template vector<XT>(w, p.w, p.w_f32, t, p.D, 0.f);
#pragma unroll
  for (int n = 0; n < S::P; ++n) acc[n] = f2(0.f);
  const float over = 1.f / p.D;
  int flip = 0, stage = 0;
  for (int turn = 0; turn < turns.all; ++turn, flip ^= 1, pdx.next(), pdz.next()) {
    const bool live = turn < turns.mine;
    Raw<XT, 8> x[S::R], z[S::R], d[S::R];
    if constexpr (Ring::kOn) {
      Ring::wait();
      ring.template take<XT, kX>(x, stage);
      ring.template take<XT, kZ>(z, stage);
      ring.template take<XT, kD>(d, stage);
      fetch(stage ? stage - 1 : Ring::kStages - 1);
      stage = stage + 1 == Ring::kStages ? 0 : stage + 1;
    }
    if (!Ring::kOn || !live) {      // (a row that is not there adds nothing)
#pragma unroll
      for (int i = 0; i < S::R; ++i) {
        x[i].zero();
        z[i].zero();
        d[i].zero();
      }
    }
    if constexpr (!Ring::kOn) {
      if (live) {
        S::template load<XT>(x, px.p, t, p.D);
        S::template load<XT>(z, pz.p, t, p.D);
        S::template load<XT>(d, pd.p, t, p.D);
      }
      next();
    }
    F2 xx = f2(0.f), dx_sum = f2(0.f), dn[S::P], slope[S::P];
#pragma unroll
    for (int n = 0; n < S::P; ++n) {
      F2 e;
      const F2 xv = x[n / 4].get2(n % 4), zv = z[n / 4].get2(n % 4), dv = d[n / 4].get2(n % 4), sg = logistic<XT>(zv, e), ds = dv * sg;
      dn[n] = SILU ? ds * zv : ds;
      slope[n] = ds * (SILU ? fma2(zv, fma2(sg, f2(-1.f), f2(1.f)), f2(1.f)) : one_less(sg, e));      // (beside the 1 of silu the subtraction does no harm)
      xx = fma2(xv, xv, xx);
      dx_sum = fma2(dn[n] * w[n], xv, dx_sum);
    }
    float s[2] = {lo(xx) + hi(xx), lo(dx_sum) + hi(dx_sum)};
    S::template row_sums<2>(s, sums[flip]);
    const float r1 = live ? rsqrtf(fmaf(s[0], over, p.eps)) : 0.f;      // (with eps = 0 a row that is not there would have an infinite root)
    const F2 r = f2(r1), c = f2(-s[1] * over * r1 * r1);
    F2 dx[S::P];
#pragma unroll
    for (int n = 0; n < S::P; ++n) {
      const F2 xv = x[n / 4].get2(n % 4), xr = xv * r;
      dx[n] = r * fma2(xv, c, dn[n] * w[n]);
      acc[n] = fma2(dn[n], xr, acc[n]);
      slope[n] = slope[n] * (xr * w[n]);
    }
    if (live) {
      if (p.dx) S::template store<XT>(dx, pdx.p, t, p.D);
      if (p.dz) S::template store<XT>(slope, pdz.p, t, p.D);
    }
  }
  if (!p.part) return;
  griddep_launch();      // (the kernel that adds the shares waits for their stores)
  S::column_share(acc, p.part + static_cast<long long>(blockIdx.x) * p.D, reinterpret_cast<float*>(smem), t, p.D);
}

// 32 columns a CTA; a warp takes every 32nd share, the warps' sums are added in their order.
template <int XT>
__global__ void __launch_bounds__(1024) column_sums_kernel(const ColumnSums c) {
  __shared__ float s[32][33];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, v = blockIdx.y, col = blockIdx.x * 32 + lane;
  float a = 0.f;
  griddep_wait();
  if (col < c.D) {
    const float* p = c.part + static_cast<long long>(v) * c.D + col;
    const long long line = static_cast<long long>(c.vectors) * c.D;
#pragma unroll 8
    for (int i = warp; i < c.parts; i += 32) a += p[i * line];
  }
  s[warp][lane] = a;
  __syncthreads();
  if (warp == 0 && col < c.D) {
    a = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) a += s[i][lane];
    if (c.f32[v]) static_cast<float*>(c.out[v])[col] = a;
    else static_cast<typename Elem<XT>::T*>(c.out[v])[col] = from_f32<XT>(a);
  }
}

int launch_column_sums(const ColumnSums& c, cudaStream_t st) {
  return by_x_type(c.x_type, [&](auto x) {
    const cudaError_t e = launch_dependent(column_sums_kernel<x.value>, dim3((c.D + 31) / 32, c.vectors), dim3(1024), 0, st, c);
    return e == cudaSuccess ? kOk : kErrLaunch;
  });
}

static int gated_problem(const LetheGdnGatedNormArgs* a, GatedProblem* p, bool backward) {
  if (!a) return kErrNull;
  if (a->rows <= 0 || a->inner <= 0 || a->inner > INT32_MAX || a->D <= 0 || a->D > kNormMaxD || !norm_types_ok(a->x_type, a->w_type) || !(a->eps >= 0.f) || !std::isfinite(a->eps)) return kErrDims;
  if (!a->x || !a->gate || !a->weight || (!backward && !a->y) || (backward && !a->dy)) return kErrNull;
  if (!on_elements(a->x_type, a->x, a->gate, a->y, a->dy, a->dx, a->dgate) || !on_elements(a->w_type, a->weight, a->dweight)) return kErrAlign;
  *p = {a->rows, a->inner, a->D, a->w_type == LETHE_F32, a->eps, a->x, a->x_outer, a->x_inner, a->gate, a->gate_outer, a->gate_inner,
        a->weight, a->y, a->dy, a->dx, a->dgate, nullptr};
  return kOk;
}

}  // namespace lg

extern "C" size_t lethe_gdn_norm_work_bytes(int64_t rows, int32_t D, int32_t vectors) {
  using namespace lg;
  if (rows <= 0 || D <= 0 || D > kNormMaxD || vectors <= 0 || vectors > 3) return 0;
  return static_cast<size_t>(std::min<int64_t>(rows, norm_parts_max(D))) * D * vectors * sizeof(float);
}

extern "C" int lethe_gdn_gated_norm(const LetheGdnGatedNormArgs* a, void* stream) {
  using namespace lg;
  GatedProblem p;
  if (int e = gated_problem(a, &p, false)) return e;
  DeviceGuard guard(a->x);
  if (!guard.ok) return kErrDevice;
  const int w = widest_piece(widest_of(a->x_type, a->x_type), p.D, [&](int n) {
    return piece_aligned(n, p.x, a->x_type, p.xo, p.xi) && piece_aligned(n, p.z, a->x_type, p.zo, p.zi) && piece_aligned(n, p.y, a->x_type);
  });
  return by_x_type(a->x_type, [&](auto x) {
    return by_row_shape<widest_of(x.value, x.value)>(p.D, w, [&](auto s) {
      using S = decltype(s);
      constexpr int smem = GatedRing<x.value, S, false>::kBytes;
      static SmemAttr attr[2];
      const auto kern = a->silu ? gated_norm_kernel<x.value, true, S> : gated_norm_kernel<x.value, false, S>;
      if (int e = attr[a->silu != 0].set(kern, smem)) return e;
      kern<<<norm_grid(p.rows, S::kRows, gated_ctas<S>(false)), S::kThreads, smem, static_cast<cudaStream_t>(stream)>>>(p);
      return launched_ok();
    });
  });
}

extern "C" int lethe_gdn_gated_norm_vjp(const LetheGdnGatedNormArgs* a, void* stream) {
  using namespace lg;
  GatedProblem p;
  if (int e = gated_problem(a, &p, true)) return e;
  if (a->dweight) {
    if (!a->work) return kErrNull;
    if (a->work_bytes < lethe_gdn_norm_work_bytes(a->rows, a->D, 1)) return kErrWorkspace;
    if (reinterpret_cast<uintptr_t>(a->work) & 15) return kErrAlign;
    p.part = static_cast<float*>(a->work);
  }
  DeviceGuard guard(a->x);
  if (!guard.ok) return kErrDevice;
  const int w = widest_piece(widest_of(a->x_type, a->x_type), p.D, [&](int n) {
    return piece_aligned(n, p.x, a->x_type, p.xo, p.xi) && piece_aligned(n, p.z, a->x_type, p.zo, p.zi) && piece_aligned(n, p.dy, a->x_type) &&
           piece_aligned(n, p.dx, a->x_type) && piece_aligned(n, p.dz, a->x_type);
  });
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int grid = 0;
  const int e = by_x_type(a->x_type, [&](auto x) {
    return by_row_shape<widest_of(x.value, x.value)>(p.D, w, [&](auto s) {
      using S = decltype(s);
      grid = std::min(norm_grid(p.rows, S::kRows, gated_ctas<S>(true)), norm_parts_max(p.D));
      constexpr int smem = std::max(GatedRing<x.value, S, true>::kBytes, S::kColumnBytes);
      static SmemAttr attr[2];
      const auto kern = a->silu ? gated_norm_vjp_kernel<x.value, true, S> : gated_norm_vjp_kernel<x.value, false, S>;
      if (int e = attr[a->silu != 0].set(kern, smem)) return e;
      kern<<<grid, S::kThreads, smem, st>>>(p);
      return launched_ok();
    });
  });
  if (e || !p.part) return e;
  return launch_column_sums({p.part, grid, 1, p.D, {a->dweight}, {p.w_f32}, a->x_type}, st);
}
