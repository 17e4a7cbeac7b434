// The element-wise gated recurrence h_t = e^{g_t} h_{t-1} + x_t (or + (1 - e^{g_t}) x_t), its backward, and one token of it.
//
// Bound by HBM: some 10 to 20 operations for every 8 bytes forward (bf16 x and h, fp32 g) and 14 backward.
//
// A tile is kTokens tokens of kChannels channels of one sequence.  A thread holds kSteps tokens of four channels in registers; its
// 16-lane group covers the channels, kGroups groups the tokens.  Two levels of the same scan: every thread runs its own tokens
// from a zero state, the groups' results (sum of g, state) meet in shared memory and are folded in order, and every thread runs
// its tokens again from the state that it really starts from.  The order of all sums is fixed, so two runs give the same bits.
//
// The decay.  With memories of thousands of tokens e^g lies next to one, and fp32 rounds it by up to 2^-25: over n tokens the
// state is off by up to n times that, always to the same side where g is constant.  So below |g| = 1/4 the step is taken with
// c = e^g - 1 from its Taylor series, h + (c h + x): c is exact to a rounding of its own, and what is left is the rounding of
// the sum, which is even.  Beyond, where a memory is a few tokens, it is e^g h + x.  Both are one fused multiply-add with a
// coefficient whose sign bit says whether h is added (c <= -0) or not (e^g >= +0).  Decays of several tokens are kept as sums of g.
#include <type_traits>

#include "elem.cuh"
#include "host_util.h"

namespace lg {

constexpr int kLanes = 16, kPer = 4, kChannels = kLanes * kPer;
constexpr int kGroups = 16, kSteps = 8, kTokens = kGroups * kSteps;
constexpr int kScanThreads = kLanes * kGroups;

// coefficient of a step over the log decay g
__device__ __forceinline__ float decay_coef(float g) {
  // e^g - 1 = g (1 + g/2 (1 + g/3 (... (1 + g/7)))): the first term left out is under 2e-9 of the result for |g| <= 1/4
  float s = fmaf(g, 1.f / 7.f, 1.f);
  s = fmaf(g * (1.f / 6.f), s, 1.f);
  s = fmaf(g * (1.f / 5.f), s, 1.f);
  s = fmaf(g * (1.f / 4.f), s, 1.f);
  s = fmaf(g * (1.f / 3.f), s, 1.f);
  s = fmaf(g * (1.f / 2.f), s, 1.f);
  const float m = __uint_as_float(__float_as_uint(g * s) | 0x80000000u);      // (g = +0 too)
  return g > -0.25f && g <= 0.f ? m : expf(g);
}
__device__ __forceinline__ bool is_diff(float c) { return static_cast<int>(__float_as_uint(c)) < 0; }
// e^g h + x
__device__ __forceinline__ float decay_step(float c, float h, float x) {
  const float t = fmaf(c, h, x);
  return is_diff(c) ? h + t : t;
}
__device__ __forceinline__ float forgotten(float c) { return is_diff(c) ? -c : 1.f - c; }      // 1 - e^g

struct DiagProblem {
  long long B, L, D;
  const void* x;
  long long x_batch, x_token;
  const void* g;
  long long g_batch, g_token;
  const float* h0;
  void* h;
  float* hT;
  float* states;
  const void* d_h;
  long long d_batch, d_token;
  const float* dhT;
  void *dx, *dg;
  float* dh0;
  int tiles, strips;      // tiles of kTokens tokens, strips of kChannels channels
};

// Four channels of one token.  VEC: neighbours, one load; else every 16th channel, element by element, D and alignment as they are.
template <bool VEC>
__device__ __forceinline__ int channel_of(int lane, int j) { return VEC ? lane * kPer + j : lane + j * kLanes; }

template <int TY, bool VEC>
__device__ __forceinline__ void load_token(Raw<TY, kPer>& r, const typename Elem<TY>::T* p, int lane, int room) {
  if constexpr (VEC) {
    if (lane * kPer < room) r.load(p + lane * kPer);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (lane + j * kLanes < room) raw_put(r, j, __ldg(p + lane + j * kLanes));
  }
}
template <int TY, bool VEC>
__device__ __forceinline__ void store_token(const Raw<TY, kPer>& r, typename Elem<TY>::T* p, int lane, int room) {
  if constexpr (VEC) {
    if (lane * kPer < room) r.store(p + lane * kPer);
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (lane + j * kLanes < room) p[lane + j * kLanes] = raw_take(r, j);
  }
}
template <int TY>
__device__ __forceinline__ Raw<TY, kPer> packed(const float (&v)[kPer]) {
  Raw<TY, kPer> r;
  r.set2(0, v[0], v[1]);
  r.set2(2, v[2], v[3]);
  return r;
}

struct ScanShared {
  float2 part[kGroups][kChannels];      // per group of tokens: (coefficient of its whole decay, state from zero)
  float start[kGroups][kChannels];      // state in front of a group
  float2 back[kGroups][kChannels];      // the same for the gradient, backwards in time
  float end[kGroups][kChannels];        // gradient that comes into a group from the tokens behind it
  float carry[2][kChannels];
};

// One CTA goes through the tiles of a strip of channels of one sequence.
template <int XT, int GT, bool VEC, bool COMP>
__global__ void __launch_bounds__(kScanThreads) diag_forward_kernel(const DiagProblem p) {
  using X = typename Elem<XT>::T;
  using G = typename Elem<GT>::T;
  __shared__ ScanShared sh;
  const int lane = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const long long b = blockIdx.x / p.strips, ch0 = static_cast<long long>(blockIdx.x % p.strips) * kChannels;
  const int room = static_cast<int>(p.D - ch0 < kChannels ? p.D - ch0 : kChannels);
  const X* x = static_cast<const X*>(p.x) + b * p.x_batch + ch0;
  const G* g = static_cast<const G*>(p.g) + b * p.g_batch + ch0;
  X* h = static_cast<X*>(p.h) + b * p.L * p.D + ch0;
  float carry = 0.f;                    // threads below kChannels: the state in front of the tile
  if (threadIdx.x < room && p.h0) carry = p.h0[b * p.D + ch0 + threadIdx.x];
  for (int tile = 0; tile < p.tiles; ++tile) {
    const long long t0 = static_cast<long long>(tile) * kTokens + grp * kSteps;
    Raw<XT, kPer> xr[kSteps];
    Raw<GT, kPer> gr[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      xr[s].zero();
      gr[s].zero();
      if (t0 + s < p.L) {
        load_token<XT, VEC>(xr[s], x + (t0 + s) * p.x_token, lane, room);
        load_token<GT, VEC>(gr[s], g + (t0 + s) * p.g_token, lane, room);
      }
    }
    float c[kSteps][kPer], sum[kPer], st[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum[j] = st[j] = 0.f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const float gv = gr[s].get(j);
        c[s][j] = decay_coef(gv);
        sum[j] += gv;
        const float u = COMP ? xr[s].get(j) * forgotten(c[s][j]) : xr[s].get(j);
        st[j] = decay_step(c[s][j], st[j], u);
      }
#pragma unroll
    for (int j = 0; j < kPer; ++j) sh.part[grp][channel_of<VEC>(lane, j)] = make_float2(decay_coef(sum[j]), st[j]);
    __syncthreads();
    if (threadIdx.x < kChannels) {
      if (p.states && threadIdx.x < room) p.states[(b * p.tiles + tile) * p.D + ch0 + threadIdx.x] = carry;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        sh.start[i][threadIdx.x] = carry;
        const float2 a = sh.part[i][threadIdx.x];
        carry = decay_step(a.x, carry, a.y);
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPer; ++j) st[j] = sh.start[grp][channel_of<VEC>(lane, j)];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const float u = COMP ? xr[s].get(j) * forgotten(c[s][j]) : xr[s].get(j);
        st[j] = decay_step(c[s][j], st[j], u);
      }
      if (t0 + s < p.L) store_token<XT, VEC>(packed<XT>(st), h + (t0 + s) * p.D, lane, room);
    }
  }
  if (threadIdx.x < room && p.hT) p.hT[b * p.D + ch0 + threadIdx.x] = carry;
}

template <int XT, int GT, bool VEC, bool COMP>
__global__ void __launch_bounds__(kScanThreads) diag_backward_kernel(const DiagProblem p) {
  using X = typename Elem<XT>::T;
  using G = typename Elem<GT>::T;
  __shared__ ScanShared sh;
  const int lane = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const long long b = blockIdx.x / p.strips, ch0 = static_cast<long long>(blockIdx.x % p.strips) * kChannels;
  const int room = static_cast<int>(p.D - ch0 < kChannels ? p.D - ch0 : kChannels);
  const X* x = static_cast<const X*>(p.x) + b * p.x_batch + ch0;
  const G* g = static_cast<const G*>(p.g) + b * p.g_batch + ch0;
  const X* d = p.d_h ? static_cast<const X*>(p.d_h) + b * p.d_batch + ch0 : nullptr;
  X* dx = p.dx ? static_cast<X*>(p.dx) + b * p.L * p.D + ch0 : nullptr;
  G* dg = p.dg ? static_cast<G*>(p.dg) + b * p.L * p.D + ch0 : nullptr;
  const int fold = threadIdx.x - kChannels;      // threads kChannels .. 2 kChannels - 1 fold the gradient
  float carry = 0.f;
  if (fold >= 0 && fold < room && p.dhT) carry = p.dhT[b * p.D + ch0 + fold];
  for (int tile = p.tiles - 1; tile >= 0; --tile) {
    const long long t0 = static_cast<long long>(tile) * kTokens + grp * kSteps;
    Raw<XT, kPer> xr[kSteps], dr[kSteps];
    Raw<GT, kPer> gr[kSteps];
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      xr[s].zero();
      gr[s].zero();
      dr[s].zero();
      if (t0 + s < p.L) {
        load_token<XT, VEC>(xr[s], x + (t0 + s) * p.x_token, lane, room);
        load_token<GT, VEC>(gr[s], g + (t0 + s) * p.g_token, lane, room);
        if (d) load_token<XT, VEC>(dr[s], d + (t0 + s) * p.d_token, lane, room);
      }
    }
    float c[kSteps][kPer], sum[kPer], st[kPer], e[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum[j] = st[j] = e[j] = 0.f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const float gv = gr[s].get(j);
        c[s][j] = decay_coef(gv);
        sum[j] += gv;
        const float u = COMP ? xr[s].get(j) * forgotten(c[s][j]) : xr[s].get(j);
        st[j] = decay_step(c[s][j], st[j], u);
      }
#pragma unroll
    for (int s = kSteps - 1; s >= 0; --s)
#pragma unroll
      for (int j = 0; j < kPer; ++j) e[j] = decay_step(c[s][j], dr[s].get(j) + e[j], 0.f);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const float whole = decay_coef(sum[j]);
      sh.part[grp][channel_of<VEC>(lane, j)] = make_float2(whole, st[j]);
      sh.back[grp][channel_of<VEC>(lane, j)] = make_float2(whole, e[j]);
    }
    __syncthreads();
    if (threadIdx.x < kChannels) {
      float s0 = threadIdx.x < room ? p.states[(b * p.tiles + tile) * p.D + ch0 + threadIdx.x] : 0.f;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        sh.start[i][threadIdx.x] = s0;
        const float2 a = sh.part[i][threadIdx.x];
        s0 = decay_step(a.x, s0, a.y);
      }
    } else if (fold < kChannels) {
#pragma unroll
      for (int i = kGroups - 1; i >= 0; --i) {
        sh.end[i][fold] = carry;
        const float2 a = sh.back[i][fold];
        carry = decay_step(a.x, carry, a.y);
      }
    }
    __syncthreads();
    float before[kSteps][kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      st[j] = sh.start[grp][channel_of<VEC>(lane, j)];
      e[j] = sh.end[grp][channel_of<VEC>(lane, j)];
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const float xv = xr[s].get(j);
        before[s][j] = COMP ? st[j] - xv : st[j];
        st[j] = decay_step(c[s][j], st[j], COMP ? xv * forgotten(c[s][j]) : xv);
      }
#pragma unroll
    for (int s = kSteps - 1; s >= 0; --s) {
      float vx[kPer], vg[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const float dv = dr[s].get(j) + e[j];
        vx[j] = COMP ? dv * forgotten(c[s][j]) : dv;
        e[j] = decay_step(c[s][j], dv, 0.f);
        vg[j] = e[j] * before[s][j];
      }
      if (t0 + s < p.L) {
        if (dx) store_token<XT, VEC>(packed<XT>(vx), dx + (t0 + s) * p.D, lane, room);
        if (dg) store_token<GT, VEC>(packed<GT>(vg), dg + (t0 + s) * p.D, lane, room);
      }
    }
  }
  if (fold >= 0 && fold < room && p.dh0) p.dh0[b * p.D + ch0 + fold] = carry;
}

struct StepProblem {
  long long B, D;
  const void* x;
  long long x_batch;
  const void* g;
  long long g_batch;
  void* h;
  float* state;
  int blocks;      // CTAs of a sequence
};

// One token: state and h, four neighbouring channels a thread (VEC) or one.
template <int XT, int GT, bool VEC, bool COMP>
__global__ void __launch_bounds__(256) diag_step_kernel(const StepProblem p) {
  using X = typename Elem<XT>::T;
  using G = typename Elem<GT>::T;
  constexpr int N = VEC ? kPer : 1;
  const long long b = blockIdx.x / p.blocks, at = (static_cast<long long>(blockIdx.x % p.blocks) * 256 + threadIdx.x) * N;
  if (at >= p.D) return;
  const X* x = static_cast<const X*>(p.x) + b * p.x_batch + at;
  const G* g = static_cast<const G*>(p.g) + b * p.g_batch + at;
  X* h = static_cast<X*>(p.h) + b * p.D + at;
  float* st = p.state + b * p.D + at;
  if constexpr (VEC) {
    Raw<XT, N> xr;
    Raw<GT, N> gr;
    xr.load(x);
    gr.load(g);
    const float4 s4 = *reinterpret_cast<const float4*>(st);
    float v[N] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float c = decay_coef(gr.get(j));
      v[j] = decay_step(c, v[j], COMP ? xr.get(j) * forgotten(c) : xr.get(j));
    }
    *reinterpret_cast<float4*>(st) = make_float4(v[0], v[1], v[2], v[3]);
    packed<XT>(v).store(h);
  } else {
    const float xv = to_f32(*x), c = decay_coef(to_f32(*g));
    const float v = decay_step(c, *st, COMP ? xv * forgotten(c) : xv);
    *st = v;
    *h = from_f32<XT>(v);
  }
}

// ---------------------------------------------------------------------------------------------
static bool types_ok(int xt, int gt) { return xt >= LETHE_F32 && xt <= LETHE_F16 && (gt == LETHE_F32 || gt == xt); }
// `n` elements of type `ty` from `ptr` on lie on a boundary of n elements, and rows `stride` apart keep to it
static bool on_boundary(const void* ptr, int ty, int n, long long s0 = 0, long long s1 = 0) {
  return reinterpret_cast<uintptr_t>(ptr) % (n * elem_bytes(ty)) == 0 && s0 % n == 0 && s1 % n == 0;
}

// f(XT, GT, VEC, COMP) as template arguments
template <typename F>
static int by_type(int xt, int gt, bool vec, bool comp, F&& f) {
  auto flags = [&](auto x, auto g) {
    if (vec) return comp ? f(x, g, std::true_type(), std::true_type()) : f(x, g, std::true_type(), std::false_type());
    return comp ? f(x, g, std::false_type(), std::true_type()) : f(x, g, std::false_type(), std::false_type());
  };
  using T32 = std::integral_constant<int, LETHE_F32>;
  using TB = std::integral_constant<int, LETHE_BF16>;
  using TH = std::integral_constant<int, LETHE_F16>;
  if (xt == LETHE_F32) return flags(T32(), T32());
  if (xt == LETHE_BF16) return gt == LETHE_F32 ? flags(TB(), T32()) : flags(TB(), TB());
  return gt == LETHE_F32 ? flags(TH(), T32()) : flags(TH(), TH());
}

static int launched() { return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch; }

static int diag_problem(const LetheGdnDiagArgs* a, DiagProblem* p, bool backward) {
  if (!a) return kErrNull;
  if (a->B <= 0 || a->L <= 0 || a->D <= 0 || !types_ok(a->x_type, a->g_type)) return kErrDims;
  if (!a->x || !a->g || !a->status || (!backward && !a->h) || (backward && !a->states)) return kErrNull;
  const long long tiles = (a->L + kTokens - 1) / kTokens, strips = (a->D + kChannels - 1) / kChannels;
  if (tiles > INT32_MAX || strips > INT32_MAX || a->B > INT32_MAX / strips) return kErrDims;
  *p = {a->B, a->L, a->D, a->x, a->x_batch, a->x_token, a->g, a->g_batch, a->g_token, a->h0, a->h, a->hT, a->states, a->d_h, a->d_h_batch,
        a->d_h_token, a->dhT, a->dx, a->dg, a->dh0, static_cast<int>(tiles), static_cast<int>(strips)};
  return kOk;
}

}  // namespace lg

extern "C" size_t lethe_gdn_diag_states_bytes(int64_t B, int64_t L, int64_t D) {
  using namespace lg;
  if (B <= 0 || L <= 0 || D <= 0) return 0;
  return static_cast<size_t>(B) * ((L + kTokens - 1) / kTokens) * D * sizeof(float);
}
extern "C" size_t lethe_gdn_diag_work_bytes(int64_t, int64_t, int64_t) { return 0; }

extern "C" int lethe_gdn_diag_forward(const LetheGdnDiagArgs* a, void* stream) {
  using namespace lg;
  DiagProblem p;
  if (int e = diag_problem(a, &p, false)) return e;
  DeviceGuard guard(a->x);
  if (!guard.ok) return kErrDevice;
  const bool vec = a->D % kPer == 0 && on_boundary(a->x, a->x_type, kPer, a->x_batch, a->x_token) &&
                   on_boundary(a->g, a->g_type, kPer, a->g_batch, a->g_token) && on_boundary(a->h, a->x_type, kPer);
  return by_type(a->x_type, a->g_type, vec, a->complement != 0, [&](auto x, auto g, auto v, auto c) {
    diag_forward_kernel<x.value, g.value, v.value, c.value>
        <<<static_cast<unsigned>(p.B * p.strips), kScanThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return launched();
  });
}

extern "C" int lethe_gdn_diag_backward(const LetheGdnDiagArgs* a, void* stream) {
  using namespace lg;
  DiagProblem p;
  if (int e = diag_problem(a, &p, true)) return e;
  DeviceGuard guard(a->x);
  if (!guard.ok) return kErrDevice;
  const bool vec = a->D % kPer == 0 && on_boundary(a->x, a->x_type, kPer, a->x_batch, a->x_token) &&
                   on_boundary(a->g, a->g_type, kPer, a->g_batch, a->g_token) &&
                   on_boundary(a->d_h, a->x_type, kPer, a->d_h_batch, a->d_h_token) && on_boundary(a->dx, a->x_type, kPer) &&
                   on_boundary(a->dg, a->g_type, kPer);
  return by_type(a->x_type, a->g_type, vec, a->complement != 0, [&](auto x, auto g, auto v, auto c) {
    diag_backward_kernel<x.value, g.value, v.value, c.value>
        <<<static_cast<unsigned>(p.B * p.strips), kScanThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return launched();
  });
}

extern "C" int lethe_gdn_diag_step(const LetheGdnDiagArgs* a, float* state, void* stream) {
  using namespace lg;
  if (!a) return kErrNull;
  if (a->B <= 0 || a->D <= 0 || !types_ok(a->x_type, a->g_type)) return kErrDims;
  if (!a->x || !a->g || !a->h || !state) return kErrNull;
  const bool vec = a->D % kPer == 0 && on_boundary(a->x, a->x_type, kPer, a->x_batch) && on_boundary(a->g, a->g_type, kPer, a->g_batch) &&
                   on_boundary(a->h, a->x_type, kPer) && on_boundary(state, LETHE_F32, kPer);
  const long long blocks = (a->D + 256 * (vec ? kPer : 1) - 1) / (256 * (vec ? kPer : 1));
  if (blocks > INT32_MAX || a->B > INT32_MAX / blocks) return kErrDims;
  DeviceGuard guard(a->x);
  if (!guard.ok) return kErrDevice;
  const StepProblem p{a->B, a->D, a->x, a->x_batch, a->g, a->g_batch, a->h, state, static_cast<int>(blocks)};
  return by_type(a->x_type, a->g_type, vec, a->complement != 0, [&](auto x, auto g, auto v, auto c) {
    diag_step_kernel<x.value, g.value, v.value, c.value>
        <<<static_cast<unsigned>(p.B * blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return launched();
  });
}
