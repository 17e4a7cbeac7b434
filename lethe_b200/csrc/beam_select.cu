// Beam search's selection.  For every group b of W beams over a vocabulary of V tokens, and T the temperature,
//
//   lse_w = log sum_v exp(l_wv / T)   over the allowed v,      c_wv = s_w + (l_wv / T - lse_w),      r_wv = c_wv / penalty_w
//
// the k largest r, of equal ones the lowest (w, v).  A finished beam offers r = s_w / penalty_w at the token eos and nothing else.
//
// What has to cross HBM is every logit, once.  Within a beam the order of r is that of the logits, whatever lse_w is, so one pass
// suffices: a warp takes a segment of a row, sums exponentials relative to the largest logit it has seen, and leaves the k largest of the
// segment among a few more, in no order (beam_scan_kernel); a CTA per group adds up the sums and merges the lists (beam_merge_kernel).
//
// Between beams candidates can be as close as they like.  The logarithms of the sums are within kLseError of the formula (below); where two candidates of
// different beams that decide the result are closer than two such errors, the merge sums the exponentials of those beams again in 64 bits.
//
// Measured, a pass through the public call: 64 x 8 x 131072 bf16, k = 16 (134 MB, 20.5 us at the copy rate) 36 us, of it the scan 30 and the merge 5;
// 16 x 8 x 65536 13 us; 1 x 4 x 32000 9 us, which is the latency of the two kernels (4 + 5).  What bounds the scan of large batches: its loads alone take
// 20.7 us, with the exponentials 24.4 (a quarter of that rate's hardware exp2 is left), the look for candidates adds 5.5.
#include <math.h>

#include <type_traits>

#include "elem.cuh"
#include "host_util.h"
#include "umma.cuh"

namespace lg {

constexpr int kBeamMost = 64;                     // beams of a group, and candidates asked for
constexpr int kTileLogits = 1024;                 // a warp takes that many at a time, a lane 32 of them
// Small CTAs, as many on an SM as their tiles in shared memory leave room for: 28 warps, each with two tiles on their way while it works on a third.
// With the tiles in registers instead (48 warps) the scan of 64 x 8 x 131072 took 35 us for 30, with a prefetch into registers 43.
constexpr int kScanWarps = 2, kScanCtas = 14;
constexpr int kMostTiles = 8;                     // of a segment; the rule is at scan_plan
constexpr int kCands = 128;                       // candidates of a segment that are looked at together
constexpr int kSpare = 16;                        // more than asked for that a list may have
__host__ __device__ constexpr int list_room(int k) { return (k + kSpare + 1) / 2 * 2; }      // keys come in pairs
constexpr int kMergeThreads = 512, kBins = 128, kMergeRoom = 2 * kMergeThreads;
constexpr int kMergeKeys = 4096;                  // of a group's lists, that are fetched before it is known which are wanted
constexpr int kBehind = 8;                        // candidates behind the last chosen one that are looked at for equals
// How far the logarithm of a beam's sum can be off.  A term: exp2 by the hardware 2^-22; its argument t is rounded three times (the difference,
// log2(e) / T, their product), 2^-24 |t| each; six roundings of sums in 32 bits.  The rest is in 64 bits.  What the arguments add to a sum, relative to it, is the
// mean of |t| weighted with 2^t.  Of n terms, one t = 0 and the others not above it, that mean m is largest with all others at t = -(m + 1 / ln 2), where
// n - 1 = ln 2 e m 2^m: 8.93 for a segment's 8192 (terms up to kSlack above what they are relative to lower it; several references of a segment,
// several segments: the worst of them).  A token far above a flat tail comes to 1.1e-6 of the 1.72e-6.
constexpr int kMostSummed = kMostTiles * kTileLogits;
static_assert(kMostSummed <= 8192, "the mean of |t| is below 9 up to here");
constexpr double kLseError = .693148 * 3 * 9 * 5.9605e-8 + 2.3842e-7 + 6 * 5.9605e-8;
constexpr float kSlack = 2.f;                     // how far (as a power of two) terms may be above what they are relative to

struct ScanStat {
  float m;          // largest logit
  int n;            // candidates in the list, the k largest of the segment among them, in no order
  double s;         // sum of exp((l - m) / T); NaN: the beam has no distribution
};

struct BeamProblem {
  const void* logits;
  long long batch, beam;                  // strides
  const uint8_t* allowed;
  long long a_batch, a_beam;
  const float *scores, *penalty;
  const uint8_t* finished;
  int B, W, k, V, eos;
  int tiles, lists;                       // of a segment; of a row
  float over;                             // log2(e) / T
  double inverse;                         // 1 / T
  ScanStat* stat;                         // [B, W, lists]
  unsigned long long* keys;               // [B, W, lists, list_room(k)]
  float* out_scores;
  long long *parents, *tokens;
  uint8_t* out_finished;
};

// Whole numbers in the order of the values they stand for.
constexpr uint32_t kLeast = 0x007fffffu;          // minus infinity
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);    // (both zeros are the same logit)
  return x == x ? ((u & 0x80000000u) ? ~u : u | 0x80000000u) : 0u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) { return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ unsigned long long ordered(double x) {
  const unsigned long long u = __double_as_longlong(x + 0.);
  return (u >> 63) ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double from_ordered(unsigned long long u) { return __longlong_as_double((u >> 63) ? u & ~(1ull << 63) : ~u); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// exp(t) for t <= 0 in 64 bits: 2^n e^f with n the nearest whole number to t / ln 2, f = t - n ln 2 by Cody and Waite's reduction (ln 2 as its value in
// 64 bits and what that leaves out), and e^f by its power series to the twelfth power (the next term is below 2^-52); what is below e^-700 is zero.
__device__ __forceinline__ double exp_below(double t) {
  t = fmax(t, -700.);
  const double n = rint(t * 1.4426950408889634), f = fma(n, -2.3190468138462996e-17, fma(n, -0.69314718055994529, t));
  double e = 1. / 479001600.;
  const double over[] = {1. / 39916800., 1. / 3628800., 1. / 362880., 1. / 40320., 1. / 5040., 1. / 720., 1. / 120., 1. / 24., 1. / 6., .5, 1., 1.};
#pragma unroll
  for (int i = 0; i < 12; ++i) e = fma(e, f, over[i]);
  return t <= -700. ? 0. : __longlong_as_double(__double_as_longlong(e) + (static_cast<long long>(n) << 52));
}

// The same by eighths of powers of two, roots[i] = 2^(i / 8): the seventh power of what is left is below 2^-43 of the result.  For many terms, so
// without conversions to and from 64 bits, which the GPU has few units for: the whole number is read off a sum with 1.5 2^52.
__device__ __forceinline__ double exp_below(double t, const double* roots) {
  constexpr double kWhole = 6755399441055744.;
  t = fmax(t, -700.);
  const double m = fma(t, 8 * 1.4426950408889634, kWhole), n = m - kWhole;
  const int k = static_cast<int>(__double2loint(m));
  const double f = fma(n, -2.3190468138462996e-17 / 8, fma(n, -0.69314718055994529 / 8, t));
  double e = 1. / 720.;
  const double over[] = {1. / 120., 1. / 24., 1. / 6., .5, 1., 1.};
#pragma unroll
  for (int i = 0; i < 6; ++i) e = fma(e, f, over[i]);
  e *= roots[k & 7];
  return t <= -700. ? 0. : __hiloint2double(__double2hiint(e) + (k >> 3) * (1 << 20), __double2loint(e));
}
// x in 64 bits, where what is below the normal numbers is zero and minus infinity some number below -2^127
__device__ __forceinline__ double widen(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x7f800000u ? __hiloint2double(static_cast<int>((u & 0x80000000u) | (((u & 0x7fffffffu) >> 3) + (896u << 20))), static_cast<int>(u << 29)) : 0.;
}

// log(s) for s >= 1 in 64 bits: what fp32 says, and log(s e^-y) = log(1 + d) behind it, d below 2^-19
__device__ __forceinline__ double log_above(double s) {
  const double y = logf(static_cast<float>(s)), d = fma(s, exp_below(-y), -1.);
  return y + (d - .5 * d * d);
}

// whether the beam goes on: one that does not offers nothing, or only itself
__device__ __forceinline__ bool counts(const BeamProblem& p, int row) {
  const float pen = p.penalty ? p.penalty[row] : 1.f;
  return isfinite(p.scores[row]) && pen > 0.f && pen < INFINITY;
}
__device__ __forceinline__ bool goes_on(const BeamProblem& p, int row) { return counts(p, row) && !(p.finished && p.finished[row]); }

__device__ __forceinline__ void fetch16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}

template <int TY> struct Row {
  using T = typename Elem<TY>::T;
  static constexpr int N = 16 / sizeof(T);        // logits of 16 bytes
  static constexpr int kVecs = 32 / N;            // of a lane and tile
  static constexpr int kDepth = N == 4 ? 2 : 3;   // tiles on their way
  using Vec = Raw<TY, N>;
  const T* x;
  const uint8_t* ok;                              // NULL: every token is allowed
  int V, past;                                    // past: elements between a 16-byte boundary and the row

  __device__ __forceinline__ Row(const BeamProblem& p, int row) {
    const int b = row / p.W, w = row % p.W;
    x = static_cast<const T*>(p.logits) + b * p.batch + w * p.beam;
    ok = p.allowed ? p.allowed + b * p.a_batch + w * p.a_beam : nullptr;
    V = p.V;
    past = static_cast<int>(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
  }
  __device__ __forceinline__ T least() const { return from_f32<TY>(-INFINITY); }
  __device__ __forceinline__ T at(int v) const { return v >= 0 && v < V && (!ok || ok[v]) ? x[v] : least(); }
  __device__ __forceinline__ bool inside(int v) const { return v >= 0 && v <= V - N; }
  __device__ __forceinline__ bool astride(int v) const { return !inside(v) && v > -N && v < V; }      // at an end of the row
  static constexpr uint32_t kNone = TY == LETHE_F32 ? 0xff800000u : TY == LETHE_BF16 ? 0xff80ff80u : 0xfc00fc00u;
  static __device__ __forceinline__ Vec none() {
    Vec r;
    r.w[0] = r.w[1] = r.w[2] = r.w[3] = kNone;
    return r;
  }
  // the mask's bytes for [v, v + N)
  struct Marks {
    uint32_t w[N / 4];
  };
  __device__ __forceinline__ Marks marks(int v) const {
    const uint8_t* const m = ok + v;
    Marks r;
    if (reinterpret_cast<uintptr_t>(ok - past) % N == 0) {      // (every v + past is a multiple of N)
#pragma unroll
      for (int i = 0; i < N / 4; ++i) r.w[i] = reinterpret_cast<const uint32_t*>(m)[i];
    } else {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) r.w[i] = m[4 * i] | m[4 * i + 1] << 8 | m[4 * i + 2] << 16 | static_cast<uint32_t>(m[4 * i + 3]) << 24;
    }
    return r;
  }
  // minus infinity in the place of what is not allowed
  static __device__ __forceinline__ void mask(Vec& r, const Marks& marks) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t b = __vcmpne4(marks.w[N == 4 ? 0 : i / 2], 0u);
      const uint32_t k = N == 4 ? __byte_perm(b, 0, i * 0x1111) : __byte_perm(b, 0, i % 2 ? 0x3322 : 0x1100);
      r.w[i] = (r.w[i] & k) | (kNone & ~k);
    }
  }
  // logits [v, v + N) at an end of the row, one by one, minus infinity in the place of what is not there or not allowed
  __device__ __forceinline__ Vec end(int v) const {
    Vec r;
#pragma unroll
    for (int i = 0; i < N; ++i) raw_put<TY, N>(r, i, at(v + i));
    return r;
  }
  // which of a lane's part of a tile are not below `floor`, one of them at least is not; the place of a bit's element
  static __device__ __forceinline__ uint32_t reaching(const Vec (&x)[kVecs], float floor) {
    uint32_t hit = 0;
    if constexpr (TY == LETHE_F32) {
#pragma unroll
      for (int i = 0; i < 32; ++i) hit |= static_cast<uint32_t>(x[i / N].get(i % N) >= floor) << i;
    } else {
      using T2 = typename std::conditional<TY == LETHE_BF16, __nv_bfloat162, __half2>::type;
      T2 f;
      if constexpr (TY == LETHE_BF16) f.x = f.y = __float2bfloat16_ru(floor);
      else f.x = f.y = __float2half_ru(floor);
#pragma unroll
      for (int i = 0; i < 16; ++i) hit |= __hge2_mask(*reinterpret_cast<const T2*>(&x[i / 4].w[i % 4]), f) & (0x10001u << i);
    }
    return hit;
  }
  static __device__ __forceinline__ int element(int bit) { return TY == LETHE_F32 ? bit : bit % 16 * 2 + bit / 16; }
  // the largest of a lane's part of a tile; NaN is none
  static __device__ __forceinline__ float largest(const Vec (&x)[kVecs]) {
    if constexpr (TY == LETHE_F32) {
      float m = x[0].get(0);
#pragma unroll
      for (int i = 1; i < 32; ++i) m = fmaxf(m, x[i / N].get(i % N));
      return fmaxf(m, -INFINITY);
    } else {
      using T2 = typename std::conditional<TY == LETHE_BF16, __nv_bfloat162, __half2>::type;
      auto two = [&](int i) { return *reinterpret_cast<const T2*>(&x[i / 4].w[i % 4]); };
      T2 m = two(0);
#pragma unroll
      for (int i = 1; i < 16; ++i) m = __hmax2(m, two(i));
      return fmaxf(fmaxf(to_f32(m.x), to_f32(m.y)), -INFINITY);
    }
  }
};

// Segment of a row: the lanes' tiles lie 16 bytes a lane beside one another, so element e of vector n of a lane is token
// first + tile kTileLogits + n 32 N + lane N + e.  A lane's part of a tile is a bin.
template <int TY, bool MASK>
__global__ void __launch_bounds__(32 * kScanWarps, TY == LETHE_F32 ? 11 : kScanCtas) beam_scan_kernel(const BeamProblem p) {
  using R = Row<TY>;
  using T = typename R::T;
  constexpr int N = R::N, kDepth = R::kDepth, kTile = R::kVecs * 32;
  __shared__ T tops[kScanWarps][kMostTiles][32];                  // maxima of the bins
  __shared__ uint4 rings[kScanWarps][kDepth * kTile];             // tiles on their way; afterwards a bin for each lane, and candidates
  static_assert(kCands * (sizeof(unsigned long long) + sizeof(uint16_t)) <= (kDepth - 1) * kTile * sizeof(uint4), "candidates lie where tiles were");
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const unsigned task = blockIdx.x * kScanWarps + warp, lists = p.lists, row = task / lists;
  griddep_wait();
  griddep_launch();      // (the merge waits for the lists)
  if (row >= static_cast<unsigned>(p.B) * p.W) return;
  const R r(p, row);
  const int first = static_cast<int>(task - row * lists) * p.tiles * kTileLogits - r.past;
  // A lane's part of a tile lies where only that lane reads it, so it waits for nobody else.
  typename R::Vec x[R::kVecs];
  uint4* const ring = rings[warp] + lane;
  auto fetch = [&](int j) {
    if (j < p.tiles) {
      uint4* const slot = ring + j % kDepth * kTile;
      const int v0 = first + j * kTileLogits, v = v0 + lane * N;
      auto copy = [&](int n) { fetch16(slot + n * 32, r.x + v + n * 32 * N); };
      if (v0 >= 0 && v0 <= r.V - kTileLogits) {
#pragma unroll
        for (int n = 0; n < R::kVecs; ++n) copy(n);
      } else {
        bool ends = false;
#pragma unroll
        for (int n = 0; n < R::kVecs; ++n) {
          if (r.inside(v + n * 32 * N)) copy(n);
          else slot[n * 32] = make_uint4(R::kNone, R::kNone, R::kNone, R::kNone);
          ends |= r.astride(v + n * 32 * N);
        }
        if (ends)
#pragma unroll 1
          for (int n = 0; n < R::kVecs; ++n)
            if (r.astride(v + n * 32 * N)) {
              const typename R::Vec y = r.end(v + n * 32 * N);
              slot[n * 32] = make_uint4(y.w[0], y.w[1], y.w[2], y.w[3]);
            }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int j = 0; j < kDepth - 1; ++j) fetch(j);
  if (!goes_on(p, row)) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    return;
  }
  // The sum of 2^t, t = (l - ref) over: ref is the warp's largest logit so far, or up to kSlack behind it.
  float ref = -INFINITY, mine = -INFINITY;
  double s = 0.;
  for (int j = 0; j < p.tiles; ++j) {
    fetch(j + kDepth - 1);
    const int v = first + j * kTileLogits + lane * N;
    typename R::Marks marks[R::kVecs];
    if (MASK)
#pragma unroll
      for (int n = 0; n < R::kVecs; ++n)
        if (r.inside(v + n * 32 * N)) marks[n] = r.marks(v + n * 32 * N);
    asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
#pragma unroll
    for (int n = 0; n < R::kVecs; ++n) {
      const uint4 y = ring[j % kDepth * kTile + n * 32];
      x[n].w[0] = y.x, x[n].w[1] = y.y, x[n].w[2] = y.z, x[n].w[3] = y.w;
      if (MASK && r.inside(v + n * 32 * N)) R::mask(x[n], marks[n]);
    }
    const float m = R::largest(x);
    tops[warp][j][lane] = from_f32<TY>(m);
    mine = fmaxf(mine, m);
    if (__any_sync(~0u, m > ref && !((m - ref) * p.over <= kSlack))) {
      const float now = from_ordered(__reduce_max_sync(~0u, ordered(m)));
      if (ref > -INFINITY) s *= exp_below((static_cast<double>(ref) - now) * p.inverse);
      ref = now;
    }
    const F2 less = f2(ref == -INFINITY ? 0.f : -ref), over = f2(p.over);
    F2 sum[4];
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      const F2 t = (x[n / (N / 2)].get2(n % (N / 2)) + less) * over;
      const F2 e = f2(ex2(lo(t)), ex2(hi(t)));
      sum[n % 4] = n < 4 ? e : sum[n % 4] + e;
    }
    const F2 t = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    s += static_cast<double>(lo(t) + hi(t));
  }
  __syncwarp();
  unsigned long long* const cand = reinterpret_cast<unsigned long long*>(rings[warp] + kTile);
  uint16_t* const passed = reinterpret_cast<uint16_t*>(cand + kCands);
  auto top_of = [&](int j) { return ordered(to_f32(tops[warp][j][lane])); };
  const uint32_t own = ordered(mine), top = __reduce_max_sync(~0u, own);

  // A logit that k bins or a few more have something as large as, by halving: what is below it is not among the k largest, and only
  // those bins have any of them.  Few candidates: by the lanes' maxima alone, which lets some more pass.
  constexpr int kMore = 4, kFew = 16;
  uint32_t least = kLeast + 1, above = top + 1;
  if (p.k <= 32) least = max(least, __reduce_min_sync(~0u, own));
  auto halve = [&](auto reach) {
    if (reach(least) <= p.k + kMore) return;
    while (above - least > 1) {
      const uint32_t mid = least + (above - least) / 2;
      const int n = reach(mid);
      if (n < p.k) {
        above = mid;
      } else {
        least = mid;
        if (n <= p.k + kMore) break;
      }
    }
  };
  if (p.k <= kFew) {
    halve([&](uint32_t u) { return __popc(__ballot_sync(~0u, own >= u)); });
  } else {
    halve([&](uint32_t u) {
      int n = 0;
      for (int j = 0; j < p.tiles; ++j) n += top_of(j) >= u;
      return static_cast<int>(__reduce_add_sync(~0u, n));
    });
  }
  // places in front of the lanes' own
  auto offset = [&](int n, int* all) {
    int a = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int b = __shfl_up_sync(~0u, a, d);
      if (lane >= d) a += b;
    }
    *all = __shfl_sync(~0u, a, 31);
    return a - n;
  };
  uint32_t hit = 0;
  if (own >= least)
#pragma unroll
    for (int j = 0; j < kMostTiles; ++j)
      if (j < p.tiles) hit |= static_cast<uint32_t>(top_of(j) >= least) << j;
  int reached, n = 0;
  int at = offset(__popc(hit), &reached);
  for (; hit; hit &= hit - 1, ++at)
    if (at < kCands) passed[at] = static_cast<uint16_t>((__ffs(hit) - 1) * 32 + lane);
  __syncwarp();
  // their logits, a bin for each lane
  const float floor = from_ordered(least);
  if (reached > kCands) n = kCands + 1;
  for (int i = 0; i == 0 || (i < reached && n <= kCands); i += 32) {
    int v = 0;
    const bool any = i + lane < reached && n <= kCands;
    if (any) {
      const int bin = passed[i + lane];
      v = first + bin / 32 * kTileLogits + bin % 32 * N;
      typename R::Marks marks[R::kVecs];
      if (v >= 0 && v <= r.V - N - (R::kVecs - 1) * 32 * N) {
#pragma unroll
        for (int b = 0; b < R::kVecs; ++b) {
          x[b].load(r.x + v + b * 32 * N);
          if (MASK) marks[b] = r.marks(v + b * 32 * N);
        }
        if (MASK)
#pragma unroll
          for (int b = 0; b < R::kVecs; ++b) R::mask(x[b], marks[b]);
      } else {
#pragma unroll
        for (int b = 0; b < R::kVecs; ++b) {
          const int u = v + b * 32 * N;
          x[b] = R::none();
          if (r.inside(u)) {
            x[b].load(r.x + u);
            if (MASK) R::mask(x[b], r.marks(u));
          }
        }
#pragma unroll 1
        for (int b = 0; b < R::kVecs; ++b)
          if (r.astride(v + b * 32 * N)) {
            const typename R::Vec y = r.end(v + b * 32 * N);
#pragma unroll
            for (int c = 0; c < R::kVecs; ++c)
              if (c == b) x[c] = y;
          }
      }
    }
    if (i == 0) {      // (while they come)
#pragma unroll
      for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
    }
    if (any) {
      hit = R::reaching(x, floor);
#pragma unroll
      for (int b = 0; b < R::kVecs; ++b) ring[b * 32] = make_uint4(x[b].w[0], x[b].w[1], x[b].w[2], x[b].w[3]);
    }
    int all;
    at = n + offset(__popc(hit), &all);
    n += all;
    for (; hit; hit &= hit - 1, ++at) {
      const int b = R::element(__ffs(hit) - 1);
      const float l = to_f32(reinterpret_cast<const T*>(ring + b / N * 32)[b % N]);
      if (at < kCands) cand[at] = static_cast<unsigned long long>(ordered(l)) << 32 | static_cast<uint32_t>(~(v + b / N * 32 * N + b % N));
    }
  }
  __syncwarp();
  unsigned long long* const list = p.keys + static_cast<long long>(task) * list_room(p.k);
  if (n <= list_room(p.k)) {
    for (int i = lane; i < n; i += 32) list[i] = cand[i];
  } else if (n <= kCands) {
    for (int i = lane; i < n; i += 32) {
      const unsigned long long c = cand[i];
      int before = 0;
      for (int j = 0; j < n; ++j) before += cand[j] > c;
      if (before < p.k) list[before] = c;
    }
    n = p.k;
  } else {
    // Too many equal ones, or large ones side by side: the largest of the segment, then the largest behind it, k times.
    unsigned long long last = ~0ull;
    for (n = 0; n < p.k; ++n) {
      unsigned long long best = 0;
      for (int j = 0; j < p.tiles * kTileLogits / 32; ++j) {
        const int v = first + j * 32 + lane;
        const uint32_t u = ordered(to_f32(r.at(v)));
        const unsigned long long c = static_cast<unsigned long long>(u) << 32 | static_cast<uint32_t>(~v);
        if (u > kLeast && c < last && c > best) best = c;
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) best = max(best, __shfl_xor_sync(~0u, best, d));
      if (!best) break;
      if (lane == 0) list[n] = best;
      last = best;
    }
  }
  if (lane == 0) {
    const float m = from_ordered(top);
    if (ref < m) s *= exp_below((static_cast<double>(ref) - m) * p.inverse);
    p.stat[task] = ScanStat{m, n, s};
  }
}

// A candidate: larger ones come first.
struct Entry {
  unsigned long long rank, place;      // ordered(r); ~(w 2^32 + v)
};
__device__ __forceinline__ bool larger(const Entry& a, const Entry& b) { return (a.rank > b.rank) | ((a.rank == b.rank) & (a.place > b.place)); }
__device__ __forceinline__ int beam_of(const Entry& e) { return static_cast<int>(~e.place >> 32); }
__device__ __forceinline__ int token_of(const Entry& e) { return static_cast<int>(~static_cast<uint32_t>(e.place)); }

struct MergeMemory {
  unsigned long long keys[kMergeKeys];
  ScanStat stat[kMergeThreads];
  Entry room[kMergeRoom], sorted[kBins];
  uint4 bins[kBins / 4];
  double score[kBeamMost], penalty[kBeamMost], lse[kBeamMost], part[kMergeThreads / 32];
  double inverse[kBeamMost];            // 1 / penalty, for how far ranks can be off; 0: the beam offers nothing
  double roots[8];
  float top[kBeamMost];
  int2 todo[kMergeThreads];             // list, beam
  uint32_t least;
  int n, lists;
  bool on[kBeamMost], ended[kBeamMost], again[kBeamMost];
};

// The largest of room[0, n), at most `most`, in order, as sorted[0, n).
__device__ __forceinline__ int sort_largest(MergeMemory& m, int most) {
  __syncthreads();
  const int n = m.n, tid = threadIdx.x;
  // as many threads for an entry as there are; they count those that are larger
  const int bits = n <= 32 ? 4 : n <= 64 ? 3 : n <= 128 ? 2 : n <= 256 ? 1 : 0, share = 1 << bits, part = tid & (share - 1);
  for (int i = tid >> bits; i < (n + 31) / 32 * 32; i += kMergeThreads >> bits) {      // (whole warps)
    const Entry e = m.room[min(i, n - 1)];
    int before = 0;
#pragma unroll 4
    for (int j = part; j < n; j += share) before += larger(m.room[j], e);
    for (int d = share / 2; d; d >>= 1) before += __shfl_xor_sync(~0u, before, d);
    if (i < n && before < most && part == 0) m.sorted[before] = e;
  }
  __syncthreads();
  return min(n, most);
}

template <int TY>
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamProblem p) {
  extern __shared__ __align__(16) unsigned char memory[];
  MergeMemory& m = *reinterpret_cast<MergeMemory*>(memory);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, row0 = blockIdx.x * p.W;
  const int lists = p.W * p.lists, most = p.k + kBehind, line = list_room(p.k);
  const double over = p.inverse;
  const ScanStat* stat = p.stat + static_cast<long long>(row0) * p.lists;
  const unsigned long long* keys = p.keys + static_cast<long long>(row0) * p.lists * line;
  if (tid < p.W) {      // (older than the scan, which has waited for what was before it when this kernel starts)
    const bool in = counts(p, row0 + tid), ended = p.finished && p.finished[row0 + tid];
    m.score[tid] = p.scores[row0 + tid];
    m.penalty[tid] = p.penalty ? p.penalty[row0 + tid] : 1.;
    m.inverse[tid] = in ? 1. / m.penalty[tid] : 0.;
    m.on[tid] = in && !ended;
    m.ended[tid] = in && ended;
    m.again[tid] = false;
  }
  const int w_of_tid = tid / p.lists;
  auto beam_of_list = [&](int l) { return l == tid ? w_of_tid : l / p.lists; };
  // (a product with 1 / penalty would be another number: 49 and 1 / 49 make less than one)
  auto ranked = [&](int w, double c) { return p.penalty ? __ddiv_rn(c, m.penalty[w]) : c; };
  auto begin = [&] {      // finished beams offer themselves
    if (tid == 0) m.n = m.lists = m.least = 0;
    if (tid < kBins / 4) m.bins[tid] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    if (tid < p.W && m.ended[tid])
      m.room[atomicAdd(&m.n, 1)] = Entry{ordered(ranked(tid, m.score[tid])), ~(static_cast<unsigned long long>(tid) << 32 | static_cast<uint32_t>(p.eos))};
  };
  begin();
  griddep_wait();
  if (lists <= kMergeThreads) {
    if (tid < lists) fetch16(&m.stat[tid], &stat[tid]);
    stat = m.stat;
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  if (lists * line <= kMergeKeys) {
    for (int i = 2 * tid; i < lists * line; i += 2 * kMergeThreads) fetch16(&m.keys[i], &keys[i]);
    keys = m.keys;
  }
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 1;" ::: "memory");
  __syncthreads();
  for (int w = warp; w < p.W; w += kMergeThreads / 32) {
    if (!m.on[w]) continue;
    const ScanStat* const a = stat + w * p.lists;
    float top = -INFINITY;
    for (int i = lane; i < p.lists; i += 32) top = fmaxf(top, a[i].m);
    top = from_ordered(__reduce_max_sync(~0u, ordered(top)));
    double s = 0.;
    for (int i = lane; i < p.lists; i += 32) {
      const ScanStat t = a[i];
      s += t.m == -INFINITY ? t.s : t.s * exp_below((static_cast<double>(t.m) - top) * over);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
    if (lane == 0) {
      m.on[w] = s > 0. && s < INFINITY && top < INFINITY;
      m.top[w] = top;
      m.lse[w] = __dmul_rn(top, over) + log_above(s);
    }
  }
  // (the products rounded by themselves: the one token of a beam that may say one only has log probability zero)
  auto rank = [&](int w, float x) { return ranked(w, m.score[w] + (__dmul_rn(x, over) - m.lse[w])); };
  auto entry = [&](int w, unsigned long long key) {
    return Entry{ordered(rank(w, from_ordered(static_cast<uint32_t>(key >> 32)))), ~(static_cast<unsigned long long>(w) << 32) ^ (~static_cast<uint32_t>(key))};
  };
  auto narrow = [](double x) { return ordered(static_cast<float>(x)); };      // in the same order, equal ones more
  int n;
  for (int pass = 0;; ++pass) {
    if (pass) begin();
    __syncthreads();
    // `least`: as many bins as candidates are wanted have a list whose largest logit reaches it.  What is below is not wanted.
    uint32_t head = 0;
    for (int l = tid; l < lists; l += kMergeThreads) {
      const int w = beam_of_list(l);
      if (m.on[w] && stat[l].n > 0) head = max(head, narrow(rank(w, stat[l].m)));
    }
    if (head) atomicMax(reinterpret_cast<uint32_t*>(m.bins) + tid % kBins, head);
    if (!pass) asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    {
      constexpr int kShare = kMergeThreads / kBins;
      const int i = tid / kShare;
      const uint32_t b = reinterpret_cast<const uint32_t*>(m.bins)[i];
      int reach = 0;
#pragma unroll
      for (int k = 0; k < kBins / 4 / kShare; ++k) {
        const uint4 o = m.bins[k * kShare + tid % kShare];
        reach += (o.x >= b) + (o.y >= b) + (o.z >= b) + (o.w >= b);
      }
#pragma unroll
      for (int d = kShare / 2; d; d >>= 1) reach += __shfl_xor_sync(~0u, reach, d);
      if (reach >= most && tid % kShare == 0) atomicMax(&m.least, b);
    }
    __syncthreads();
    const uint32_t floor = max(m.least, 1u);
    for (int l = tid; l < lists; l += kMergeThreads) {
      const int w = beam_of_list(l);
      if (m.on[w] && stat[l].n > 0 && (lists <= kMergeThreads ? head : narrow(rank(w, stat[l].m))) >= floor) {
        const int at = atomicAdd(&m.lists, 1);
        if (at < kMergeThreads) m.todo[at] = make_int2(l, w);
      }
    }
    __syncthreads();
    // their candidates that reach it, of two lists at a time
    for (int i = warp; i < min(m.lists, kMergeThreads); i += kMergeThreads / 16) {
      const int2 a = m.todo[i], b = i + kMergeThreads / 32 < min(m.lists, kMergeThreads) ? m.todo[i + kMergeThreads / 32] : make_int2(-1, 0);
      const int an = stat[a.x].n, bn = b.x >= 0 ? stat[b.x].n : 0;
      for (int c = lane; c < max(an, bn); c += 32) {
        unsigned long long ak = 0, bk = 0;
        if (c < an) ak = keys[static_cast<long long>(a.x) * line + c];
        if (c < bn) bk = keys[static_cast<long long>(b.x) * line + c];
        auto put = [&](int w, unsigned long long key) {
          const Entry e = entry(w, key);
          if (narrow(from_ordered(e.rank)) < floor) return;
          const int at = atomicAdd(&m.n, 1);
          if (at < kMergeRoom) m.room[at] = e;
        };
        if (c < an) put(a.y, ak);
        if (c < bn) put(b.y, bk);
      }
    }
    __syncthreads();
    if (m.lists > kMergeThreads || m.n > kMergeRoom) {
      // So many equal ones: all candidates in turn, as many at a time as there is room for, and no more of those below the last wanted one.
      Entry least{0, 0};
      __syncthreads();
      begin();
      __syncthreads();
      const long long all = static_cast<long long>(lists) * line;
      for (long long i = 0; i < all; i += kMergeThreads) {
        const int l = static_cast<int>((i + tid) / line), c = static_cast<int>((i + tid) % line);
        if (l < lists && m.on[l / p.lists] && c < stat[l].n) {
          const Entry e = entry(l / p.lists, keys[static_cast<long long>(l) * line + c]);
          if (!larger(least, e)) m.room[atomicAdd(&m.n, 1)] = e;
        }
        __syncthreads();
        if (m.n > kMergeRoom - kMergeThreads) {
          const int left = sort_largest(m, most);
          if (tid < left) m.room[tid] = m.sorted[tid];
          if (tid == 0) m.n = left;
          if (left == most) least = m.sorted[most - 1];
        }
        __syncthreads();
      }
    }
    n = sort_largest(m, most);
    if (pass) break;
    // Candidates of different beams next to one another, closer than the sums are known.
    bool close = false;
    if (tid < n && tid < p.k) {
      const Entry a = m.sorted[tid];
      const int u = beam_of(a);
      double far = 1.;
      if (p.penalty)
        for (int w = 0; w < p.W; ++w) far = fmax(w ? far : 0., m.inverse[w]);
      far *= 2. * kLseError;
      int j = tid + 1;
      for (; j < n; ++j) {
        const double gap = from_ordered(a.rank) - from_ordered(m.sorted[j].rank);
        if (!(gap < far)) break;
        const int w = beam_of(m.sorted[j]);
        // (sums that differ may be rounded to the same; finished beams have none)
        if (u != w && gap < kLseError * ((m.on[u] ? m.inverse[u] : 0.) + (m.on[w] ? m.inverse[w] : 0.))) m.again[u] = m.again[w] = close = true;
      }
      // as many equals behind the last of this beam's: another beam's may lie behind them
      if (j == most && p.W > 1) {
        for (int w = 0; w < p.W; ++w) m.again[w] = true;
        close = true;
      }
    }
    if (tid < 8) m.roots[tid] = exp2(tid / 8.);
    if (!__syncthreads_or(close)) break;
    for (int w = 0; w < p.W; ++w) {
      if (!m.again[w] || !m.on[w]) continue;
      const Row<TY> r(p, row0 + w);
      double s = 0.;
      constexpr int kAhead = 8;      // (by the token's number, wherever the row lies: equal rows have equal sums)
      for (int v = tid; v < p.V; v += kAhead * kMergeThreads) {
        float x[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {      // (no branch around a load: they are under way together)
          const int u = min(v + i * kMergeThreads, p.V - 1);
          const float l = to_f32(r.x[u]);
          const bool in = (u == v + i * kMergeThreads) & (r.ok ? r.ok[u] != 0 : true);
          x[i] = in ? l : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) s += exp_below((widen(x[i]) - m.top[w]) * over, m.roots);
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
      if (lane == 0) m.part[warp] = s;
      __syncthreads();
      if (tid == 0) {
        s = 0.;
        for (int i = 0; i < kMergeThreads / 32; ++i) s += m.part[i];
        m.lse[w] = __dmul_rn(m.top[w], over) + log_above(s);
      }
      __syncthreads();
    }
  }
  if (tid < p.k) {
    const long long o = static_cast<long long>(blockIdx.x) * p.k + tid;
    const bool there = tid < n;
    const Entry e = m.sorted[tid];
    const int w = there ? beam_of(e) : 0, v = there ? token_of(e) : max(p.eos, 0);
    p.out_scores[o] = there ? static_cast<float>(from_ordered(e.rank) * m.penalty[w]) : -INFINITY;
    p.parents[o] = w;
    p.tokens[o] = v;
    if (p.out_finished) p.out_finished[o] = !there || v == p.eos || m.ended[w];
  }
}

struct ScanPlan {
  int tiles;
  long long lists, tasks;
};
// Segments as long as they can be with a warp for each on the GPU at once, up to kMostTiles; more bins than candidates in each.  Every list costs
// its look for candidates, so one tile each is too short, and longer ones than 8 leave too little to share out.  Passes in us with 1, 2, 4, 6, 8 tiles:
// 64 x 8 x 131072 78, 53, 41, 42, 36 (chosen: 8; an earlier form with 14 and 26: 49, 60); 16 x 8 x 65536 15.8, 13.5, 13.0, 14.8, 13.4 (2).
// A row that does not begin on a 16-byte boundary may reach into one more tile.  "At once" is counted with a B200's 148 SMs, whatever GPU is current, and with the CTAs of
// 16-bit types, since the workspace has to be the same wherever it is asked for: fp32 rows, 11 CTAs an SM, with 3256 to 4144 segments take a second wave.
static ScanPlan scan_plan(long long B, int W, long long V, int k, int ty, bool aligned) {
  const long long past = aligned ? 0 : 16 / elem_bytes(ty) - 1, row = (V + past + kTileLogits - 1) / kTileLogits;
  const long long even = (V + kTileLogits - 1) / kTileLogits, held = 148 * kScanWarps * kScanCtas / (B * W);      // (for every row)
  const long long most = kMostTiles, want = held ? (even + held - 1) / held : most;
  ScanPlan s;
  s.tiles = static_cast<int>(want < most ? want : most);
  if (s.tiles * 32 < k) s.tiles = (k + 31) / 32;
  s.lists = (row + s.tiles - 1) / s.tiles;
  s.tiles = static_cast<int>((row + s.lists - 1) / s.lists);
  if (s.tiles * 32 < k) s.tiles = (k + 31) / 32;
  s.tasks = B * W * s.lists;
  return s;
}
static bool beam_sizes(long long B, int W, long long V, int k, int ty) {
  return B > 0 && W > 0 && W <= kBeamMost && k > 0 && k <= kBeamMost && V > 0 && V <= (1ll << 30) && B <= (1ll << 24) && B * W <= (1ll << 24) &&
         ty >= LETHE_F32 && ty <= LETHE_F16 && B * W * ((V + 7) / kTileLogits + 1) < (1ll << 31);
}

// Whether a result lies where another group's input may still be read.  A group's CTA has its own in shared memory before it writes anything, so with as
// many candidates as beams new scores may take the place of the old ones, and the same with marks.
static bool beam_meets(const LetheGdnBeamArgs& a) {
  struct Part {
    const void* at;
    long long bytes;
    int e;
  };
  const long long beams = a.B * a.W, n = a.B * a.k;
  const Part part[] = {{a.out_scores, 4 * n, 4}, {a.out_finished, n, 1}, {a.parents, 8 * n, 8}, {a.tokens, 8 * n, 8},
                       {a.scores, 4 * beams, 4}, {a.penalty, 4 * beams, 4}, {a.finished, beams, 1}};
  const long long work = static_cast<long long>(lethe_gdn_beam_work_bytes(a.B, a.W, a.V, a.k, a.x_type));
  for (int i = 0; i < 7; ++i) {
    if (!part[i].at) continue;
    if (meet(part[i].at, part[i].bytes, a.work, work)) return true;
    for (int j = i + 1; i < 4 && j < 7; ++j) {
      const bool own = j >= 4 && part[i].at == part[j].at && part[i].e == part[j].e && a.k == a.W;
      if (part[j].at && !own && meet(part[i].at, part[i].bytes, part[j].at, part[j].bytes)) return true;
    }
  }
  return false;
}

template <int TY>
static int launch_beam(const BeamProblem& p, long long tasks, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>((tasks + kScanWarps - 1) / kScanWarps));
  if (launch_dependent(p.allowed ? beam_scan_kernel<TY, true> : beam_scan_kernel<TY, false>, grid, dim3(32 * kScanWarps), 0, st, p) != cudaSuccess) return kErrLaunch;
  static SmemAttr attr;
  if (attr.set(beam_merge_kernel<TY>, sizeof(MergeMemory))) return kErrLaunch;
  return launch_dependent(beam_merge_kernel<TY>, dim3(p.B), dim3(kMergeThreads), sizeof(MergeMemory), st, p) == cudaSuccess ? kOk : kErrLaunch;
}

}  // namespace lg

extern "C" size_t lethe_gdn_beam_work_bytes(int64_t B, int32_t W, int64_t V, int32_t k, int32_t x_type) {
  using namespace lg;
  if (!beam_sizes(B, W, V, k, x_type)) return 0;
  return static_cast<size_t>(scan_plan(B, W, V, k, x_type, false).tasks) * (sizeof(ScanStat) + 8 * static_cast<size_t>(list_room(k)));
}

extern "C" int lethe_gdn_beam_select(const LetheGdnBeamArgs* a, void* stream) {
  using namespace lg;
  if (!a || !a->logits || !a->scores || !a->out_scores || !a->parents || !a->tokens) return kErrNull;
  if (!beam_sizes(a->B, a->W, a->V, a->k, a->x_type)) return kErrDims;
  if (a->eos < -1 || a->eos >= a->V || (a->eos < 0 && (a->finished || a->out_finished))) return kErrDims;
  if (!(a->temperature >= 1e-6 && a->temperature <= 1e6)) return kErrDims;
  if (!on_elements(a->x_type, a->logits) || !on_elements(LETHE_F32, a->scores, a->penalty, a->out_scores)) return kErrAlign;
  if ((reinterpret_cast<uintptr_t>(a->parents) | reinterpret_cast<uintptr_t>(a->tokens)) % 8) return kErrAlign;
  if (!a->work) return kErrNull;
  if (reinterpret_cast<uintptr_t>(a->work) % 16) return kErrAlign;
  const int e = elem_bytes(a->x_type);
  const bool aligned = (reinterpret_cast<uintptr_t>(a->logits) | static_cast<uintptr_t>(a->logits_batch * e) | static_cast<uintptr_t>(a->logits_beam * e)) % 16 == 0;
  const ScanPlan plan = scan_plan(a->B, a->W, a->V, a->k, a->x_type, aligned);
  if (a->work_bytes < lethe_gdn_beam_work_bytes(a->B, a->W, a->V, a->k, a->x_type)) return kErrWorkspace;
  if (beam_meets(*a)) return kErrShared;
  DeviceGuard guard(a->logits);
  if (!guard.ok) return kErrDevice;
  BeamProblem p;
  p.logits = a->logits;
  p.batch = a->logits_batch;
  p.beam = a->logits_beam;
  p.allowed = a->allowed;
  p.a_batch = a->allowed_batch;
  p.a_beam = a->allowed_beam;
  p.scores = a->scores;
  p.penalty = a->penalty;
  p.finished = a->finished;
  p.B = static_cast<int>(a->B);
  p.W = a->W;
  p.k = a->k;
  p.V = static_cast<int>(a->V);
  p.eos = static_cast<int>(a->eos);
  p.tiles = plan.tiles;
  p.lists = static_cast<int>(plan.lists);
  p.inverse = 1. / a->temperature;
  p.over = static_cast<float>(1.4426950408889634 / a->temperature);
  p.stat = static_cast<ScanStat*>(a->work);
  p.keys = reinterpret_cast<unsigned long long*>(p.stat + plan.tasks);
  p.out_scores = a->out_scores;
  p.parents = reinterpret_cast<long long*>(a->parents);
  p.tokens = reinterpret_cast<long long*>(a->tokens);
  p.out_finished = a->out_finished;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a->x_type) {
    case LETHE_F32: return launch_beam<LETHE_F32>(p, plan.tasks, st);
    case LETHE_BF16: return launch_beam<LETHE_BF16>(p, plan.tasks, st);
    default: return launch_beam<LETHE_F16>(p, plan.tasks, st);
  }
}
