// Beam search's selection.  For every group b of W beams over a vocabulary of V tokens, and T the temperature,
//
//   lse_w = log sum_v exp(l_wv / T)   over the allowed v,      c_wv = s_w + (l_wv / T - lse_w),      r_wv = c_wv / penalty_w
//
// the k largest r, of equal ones the lowest (w, v).  A finished beam offers r = s_w / penalty_w at the token eos and nothing else.
//
// What has to cross HBM is every logit, once.  Within a beam the order of r is that of the logits, whatever lse_w is, so one pass
// suffices: a warp takes a segment of a row, sums exponentials relative to its own maxima, and leaves the k largest logits
// of the segment in order (beam_scan_kernel); a CTA per group adds up the sums and merges the lists (beam_merge_kernel).
//
// Between beams candidates can be as close as they like.  The sums are within kLseError of the formula (below); where two candidates of
// different beams that decide the result are closer than two such errors, the merge sums the exponentials of those beams again in 64 bits.
#include <math.h>

#include <type_traits>

#include "elem.cuh"
#include "host_util.h"
#include "umma.cuh"

namespace lg {

constexpr int kBeamMost = 64;                     // beams of a group, and candidates asked for
constexpr int kTileLogits = 1024, kMostTiles = 16; // a warp takes that many logits at a time, and so many times
constexpr int kScanWarps = 4;
constexpr int kCands = 128;                       // candidates of a segment that are looked at together
constexpr int kSpare = 16;                        // more than asked for that a list may have
constexpr int kMergeThreads = 512, kBins = 128, kMergeRoom = 2 * kMergeThreads;
constexpr int kBehind = 8;                        // candidates behind the last chosen one that are looked at for equals
// A term of a sum: exp2 by the hardware 2^-22; its argument t has two roundings of |t| 2^-24, which count with 2^t relative to the
// largest term, |t| up to kSlack there, together below 2^-22; seven roundings of sums in 32 bits.  The rest is in 64 bits.
constexpr double kLseError = 2 * 2.4e-7 + 7 * 6e-8;
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
  unsigned long long* keys;               // [B, W, lists, k + kSpare]
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

// exp(t) for t <= 0 in 64 bits: 2^n e^f with n the nearest whole number to t / ln 2, and e^f by its power series to the twelfth power (the
// next term is below 2^-52); what is below e^-700 is zero.
__device__ __forceinline__ double exp_below(double t) {
  t = fmax(t, -700.);
  const double n = rint(t * 1.4426950408889634), f = fma(n, -2.3190468138462996e-17, fma(n, -0.69314718055994529, t));
  double e = 1. / 479001600.;
  const double over[] = {1. / 39916800., 1. / 3628800., 1. / 362880., 1. / 40320., 1. / 5040., 1. / 720., 1. / 120., 1. / 24., 1. / 6., .5, 1., 1.};
#pragma unroll
  for (int i = 0; i < 12; ++i) e = fma(e, f, over[i]);
  return t <= -700. ? 0. : __longlong_as_double(__double_as_longlong(e) + (static_cast<long long>(n) << 52));
}

// whether the beam goes on: one that does not offers nothing, or only itself
__device__ __forceinline__ bool counts(const BeamProblem& p, int row) {
  const float pen = p.penalty ? p.penalty[row] : 1.f;
  return isfinite(p.scores[row]) && pen > 0.f && pen < INFINITY;
}
__device__ __forceinline__ bool goes_on(const BeamProblem& p, int row) { return counts(p, row) && !(p.finished && p.finished[row]); }

template <int TY> struct Row {
  using T = typename Elem<TY>::T;
  static constexpr int N = 16 / sizeof(T);        // logits of 16 bytes
  static constexpr int kVecs = 32 / N;            // of a lane and tile
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
  // minus infinity in the place of what is not allowed of [v, v + N)
  __device__ __forceinline__ void mask(Vec& r, int v) const {
    const uint8_t* const m = ok + v;
    uint32_t keep[N / 4];                         // a byte of ones for each allowed token
    if (reinterpret_cast<uintptr_t>(m) % N == 0) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) keep[i] = __vcmpne4(reinterpret_cast<const uint32_t*>(m)[i], 0u);
    } else {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) keep[i] = __vcmpne4(m[4 * i] | m[4 * i + 1] << 8 | m[4 * i + 2] << 16 | static_cast<uint32_t>(m[4 * i + 3]) << 24, 0u);
    }
    constexpr uint32_t kNone = TY == LETHE_F32 ? 0xff800000u : TY == LETHE_BF16 ? 0xff80ff80u : 0xfc00fc00u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t k = N == 4 ? __byte_perm(keep[0], 0, i * 0x1111) : __byte_perm(keep[i / 2], 0, i % 2 ? 0x3322 : 0x1100);
      r.w[i] = (r.w[i] & k) | (kNone & ~k);
    }
  }
  // logits [v, v + N), minus infinity in the place of what is not there or not allowed; v + past is a multiple of N
  template <bool MASK> __device__ __forceinline__ Vec load(int v) const {
    Vec r;
    if (v >= 0 && v <= V - N) {
      r.load(x + v);
      if (MASK) mask(r, v);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) raw_put<TY, N>(r, i, at(v + i));
    }
    return r;
  }
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
template <int TY> constexpr int scan_ctas(bool mask) { return TY == LETHE_F32 ? 8 : mask ? 10 : 12; }
template <int TY, bool MASK>
__global__ void __launch_bounds__(32 * kScanWarps, scan_ctas<TY>(MASK)) beam_scan_kernel(const BeamProblem p) {
  using R = Row<TY>;
  constexpr int N = R::N;
  __shared__ uint32_t tops[kScanWarps][kMostTiles][32];           // maxima of the bins
  __shared__ unsigned long long cands[kScanWarps][kCands];
  __shared__ uint16_t passed[kScanWarps][kCands];
  griddep_launch();      // (the merge waits for the lists)
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const unsigned task = blockIdx.x * kScanWarps + warp, lists = p.lists, row = task / lists;
  if (row >= static_cast<unsigned>(p.B) * p.W) return;
  if (!goes_on(p, row)) return;
  const R r(p, row);
  const int first = static_cast<int>(task - row * lists) * p.tiles * kTileLogits - r.past;

  // The sum of 2^t, t = (l - ref) over: ref is the warp's largest logit so far, or up to kSlack behind it.
  float ref = -INFINITY, mine = -INFINITY;
  double s = 0.;
  for (int j = 0; j < p.tiles; ++j) {
    typename R::Vec x[R::kVecs];
    const int v0 = first + j * kTileLogits;
    if (v0 >= 0 && v0 <= r.V - kTileLogits) {
#pragma unroll
      for (int n = 0; n < R::kVecs; ++n) x[n].load(r.x + v0 + (n * 32 + lane) * N);
      if (MASK) {
#pragma unroll
        for (int n = 0; n < R::kVecs; ++n) r.mask(x[n], v0 + (n * 32 + lane) * N);
      }
    } else {
#pragma unroll
      for (int n = 0; n < R::kVecs; ++n) x[n] = r.template load<MASK>(v0 + (n * 32 + lane) * N);
    }
    const float m = R::largest(x);
    tops[warp][j][lane] = ordered(m);
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
#pragma unroll
  for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
  const uint32_t own = ordered(mine), top = __reduce_max_sync(~0u, own);

  // A logit that k bins or a few more have something as large as, by halving: what is below it is not among the k largest, and only
  // those bins have any of them.  Few candidates: by the lanes' maxima alone, which lets some more pass.
  constexpr int kMore = 4, kFew = 16;
  uint32_t least = kLeast + 1, above = top + 1;
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
      for (int j = 0; j < p.tiles; ++j) n += tops[warp][j][lane] >= u;
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
    for (int j = 0; j < p.tiles; ++j) hit |= static_cast<uint32_t>(tops[warp][j][lane] >= least) << j;
  int reached, n = 0;
  int at = offset(__popc(hit), &reached);
  for (; hit; hit &= hit - 1, ++at)
    if (at < kCands) passed[warp][at] = static_cast<uint16_t>((__ffs(hit) - 1) * 32 + lane);
  __syncwarp();
  // their logits, a bin for each lane
  unsigned long long* const cand = cands[warp];
  const float floor = from_ordered(least);
  if (reached > kCands) {
    n = kCands + 1;
  } else {
    for (int i = 0; i < reached; i += 32) {
      int v = 0;
      if (i + lane < reached) {
        const int bin = passed[warp][i + lane];
        v = first + bin / 32 * kTileLogits + bin % 32 * N;
#pragma unroll
        for (int b = 0; b < R::kVecs; ++b) {
          const typename R::Vec x = r.template load<MASK>(v + b * 32 * N);
#pragma unroll
          for (int e = 0; e < N; ++e) hit |= static_cast<uint32_t>(x.get(e) >= floor) << (b * N + e);
        }
      }
      int all;
      at = n + offset(__popc(hit), &all);
      n += all;
      for (; hit; hit &= hit - 1, ++at) {
        const int b = __ffs(hit) - 1, u = v + b / N * 32 * N + b % N;
        if (at < kCands) cand[at] = static_cast<unsigned long long>(ordered(to_f32(r.x[u]))) << 32 | static_cast<uint32_t>(~u);
      }
    }
  }
  __syncwarp();
  unsigned long long* const list = p.keys + static_cast<long long>(task) * (p.k + kSpare);
  if (n <= p.k + kSpare) {
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
    if (ref > -INFINITY) s *= exp_below((static_cast<double>(ref) - m) * p.inverse);
    p.stat[task] = ScanStat{m, n, s};
  }
}

// A candidate: larger ones come first.
struct Entry {
  unsigned long long rank, place;      // ordered(r); ~(w V + v)
};
__device__ __forceinline__ bool larger(const Entry& a, const Entry& b) { return a.rank > b.rank || (a.rank == b.rank && a.place > b.place); }

struct MergeMemory {
  Entry room[kMergeRoom], sorted[kBins];
  double score[kBeamMost], inverse[kBeamMost], lse[kBeamMost], part[kMergeThreads / 32];      // inverse: 1 / penalty
  float top[kBeamMost];
  uint32_t bins[kBins], least;
  int todo[kMergeThreads];
  bool on[kBeamMost], ended[kBeamMost], again[kBeamMost];
  int n, lists, any;
};

// The largest of room[0, n), at most `most`, in order; `least` becomes the last of them where there are so many.
__device__ __forceinline__ void keep_largest(MergeMemory& m, int most, Entry* least) {
  __syncthreads();
  const int n = m.n, tid = threadIdx.x;
  if (n <= kMergeThreads / 8) {
    const int i = tid / 8;
    const Entry e = m.room[min(i, n - 1 < 0 ? 0 : n - 1)];
    int before = 0;
    for (int j = tid % 8; j < n; j += 8) before += larger(m.room[j], e);
#pragma unroll
    for (int d = 4; d; d >>= 1) before += __shfl_xor_sync(~0u, before, d);
    if (i < n && before < most && tid % 8 == 0) m.sorted[before] = e;
  } else {
    for (int i = tid; i < n; i += kMergeThreads) {
      const Entry e = m.room[i];
      int before = 0;
      for (int j = 0; j < n; ++j) before += larger(m.room[j], e);
      if (before < most) m.sorted[before] = e;
    }
  }
  __syncthreads();
  const int left = min(n, most);
  for (int i = tid; i < left; i += kMergeThreads) m.room[i] = m.sorted[i];
  if (tid == 0) m.n = left;
  if (left == most) *least = m.sorted[most - 1];
  __syncthreads();
}

template <int TY>
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamProblem p) {
  __shared__ MergeMemory m;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, row0 = blockIdx.x * p.W;
  const int lists = p.W * p.lists, most = p.k + kBehind, line = p.k + kSpare;
  const double over = p.inverse;
  const ScanStat* const stat = p.stat + static_cast<long long>(row0) * p.lists;
  const unsigned long long* const keys = p.keys + static_cast<long long>(row0) * p.lists * line;
  if (tid < p.W) {
    const bool in = counts(p, row0 + tid), ended = p.finished && p.finished[row0 + tid];
    m.score[tid] = p.scores[row0 + tid];
    m.inverse[tid] = in ? (p.penalty ? 1. / p.penalty[row0 + tid] : 1.) : 0.;
    m.on[tid] = in && !ended;
    m.ended[tid] = in && ended;
    m.again[tid] = false;
  }
  __syncthreads();
  griddep_wait();
  for (int w = warp; w < p.W; w += kMergeThreads / 32) {
    if (!m.on[w]) continue;
    const ScanStat* const a = stat + w * p.lists;
    float top = -INFINITY;
    for (int i = lane; i < p.lists; i += 32) top = fmaxf(top, a[i].m);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
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
      m.lse[w] = top * over + log(s);
    }
  }
  auto rank = [&](int w, float x) { return (m.score[w] + (x * over - m.lse[w])) * m.inverse[w]; };
  auto entry = [&](int l, unsigned long long key) {
    const int w = l / p.lists;
    return Entry{ordered(rank(w, from_ordered(static_cast<uint32_t>(key >> 32)))),
                 ~(static_cast<unsigned long long>(w) * p.V + (~static_cast<uint32_t>(key)))};
  };
  auto narrow = [](double x) { return ordered(static_cast<float>(x)); };      // in the same order, equal ones more
  for (int pass = 0;; ++pass) {
    __syncthreads();
    if (tid == 0) m.n = m.lists = m.least = 0;
    if (tid < kBins) m.bins[tid] = 0;
    __syncthreads();
    if (tid < p.W && m.ended[tid])
      m.room[atomicAdd(&m.n, 1)] = Entry{ordered(m.score[tid] * m.inverse[tid]), ~(static_cast<unsigned long long>(tid) * p.V + p.eos)};
    // `least`: as many bins as candidates are wanted have a list whose largest logit reaches it.  What is below is not wanted.
    uint32_t head = 0;
    for (int l = tid; l < lists; l += kMergeThreads)
      if (m.on[l / p.lists] && stat[l].n > 0) head = max(head, narrow(rank(l / p.lists, stat[l].m)));
    if (head) atomicMax(&m.bins[tid % kBins], head);
    __syncthreads();
    {
      constexpr int kShare = kMergeThreads / kBins;
      const int i = tid / kShare;
      const uint32_t b = m.bins[i];
      int before = 0;
#pragma unroll 8
      for (int j = tid % kShare; j < kBins; j += kShare) before += m.bins[j] > b || (m.bins[j] == b && j < i);
#pragma unroll
      for (int d = kShare / 2; d; d >>= 1) before += __shfl_xor_sync(~0u, before, d);
      if (before == most - 1 && tid % kShare == 0) m.least = b;
    }
    __syncthreads();
    const uint32_t floor = max(m.least, 1u);
    for (int l = tid; l < lists; l += kMergeThreads)
      if (m.on[l / p.lists] && stat[l].n > 0 && narrow(rank(l / p.lists, stat[l].m)) >= floor) {
        const int at = atomicAdd(&m.lists, 1);
        if (at < kMergeThreads) m.todo[at] = l;
      }
    __syncthreads();
    // their candidates that reach it
    for (int i = warp; i < min(m.lists, kMergeThreads); i += kMergeThreads / 32) {
      const int l = m.todo[i], n = stat[l].n;
      for (int c = lane; c < n; c += 32) {
        const Entry e = entry(l, keys[static_cast<long long>(l) * line + c]);
        if (narrow(from_ordered(e.rank)) >= floor) {
          const int at = atomicAdd(&m.n, 1);
          if (at < kMergeRoom) m.room[at] = e;
        }
      }
    }
    __syncthreads();
    Entry least{0, 0};
    if (m.lists > kMergeThreads || m.n > kMergeRoom) {
      // So many equal ones: all candidates in turn, as many at a time as there is room for.
      __syncthreads();
      if (tid == 0) m.n = 0;
      __syncthreads();
      if (tid < p.W && m.ended[tid])
        m.room[atomicAdd(&m.n, 1)] = Entry{ordered(m.score[tid] * m.inverse[tid]), ~(static_cast<unsigned long long>(tid) * p.V + p.eos)};
      const long long all = static_cast<long long>(lists) * line;
      for (long long i = 0; i < all; i += kMergeThreads) {
        const int l = static_cast<int>((i + tid) / line), c = static_cast<int>((i + tid) % line);
        if (l < lists && m.on[l / p.lists] && c < stat[l].n) {
          const Entry e = entry(l, keys[static_cast<long long>(l) * line + c]);
          if (!larger(least, e)) m.room[atomicAdd(&m.n, 1)] = e;
        }
        __syncthreads();
        const int n = m.n;
        __syncthreads();
        if (n > kMergeRoom - kMergeThreads) keep_largest(m, most, &least);
      }
    }
    keep_largest(m, most, &least);
    if (pass) break;
    // Candidates of different beams next to one another, closer than the sums are known.
    if (tid == 0) m.any = 0;
    __syncthreads();
    const int n = m.n;
    auto beam = [&](const Entry& e) { return static_cast<int>(~e.place / p.V); };
    if (tid < n && tid < p.k) {
      const Entry a = m.sorted[tid];
      const int u = beam(a);
      double far = 0.;
      if (p.penalty) {
        for (int w = 0; w < p.W; ++w) far = fmax(far, m.inverse[w]);
      } else {
        far = 1.;
      }
      far *= 2. * kLseError;
      int j = tid + 1;
      for (; j < n; ++j) {
        const double gap = from_ordered(a.rank) - from_ordered(m.sorted[j].rank);
        if (!(gap < far)) break;
        const int w = beam(m.sorted[j]);
        if (gap > 0. && u != w && gap < kLseError * (m.inverse[u] + m.inverse[w])) m.again[u] = m.again[w] = m.any = 1;
      }
      // as many equals behind the last of this beam's: another beam's may lie behind them
      if (j == most && p.W > 1) {
        for (int w = 0; w < p.W; ++w) m.again[w] = true;
        m.any = 1;
      }
    }
    __syncthreads();
    if (!m.any) break;
    for (int w = 0; w < p.W; ++w) {
      if (!m.again[w] || !m.on[w]) continue;
      const Row<TY> r(p, row0 + w);
      double s = 0.;
#pragma unroll 4
      for (int v = tid; v < p.V; v += kMergeThreads) s += exp_below((static_cast<double>(to_f32(r.at(v))) - m.top[w]) * over);
#pragma unroll
      for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
      if (lane == 0) m.part[warp] = s;
      __syncthreads();
      if (tid == 0) {
        s = 0.;
        for (int i = 0; i < kMergeThreads / 32; ++i) s += m.part[i];
        m.lse[w] = m.top[w] * over + log(s);
      }
      __syncthreads();
    }
  }
  if (tid < p.k) {
    const long long o = static_cast<long long>(blockIdx.x) * p.k + tid;
    const bool there = tid < m.n;
    const unsigned long long place = there ? ~m.sorted[tid].place : 0;
    const int w = static_cast<int>(place / p.V), v = there ? static_cast<int>(place % p.V) : max(p.eos, 0);
    p.out_scores[o] = there ? static_cast<float>(from_ordered(m.sorted[tid].rank) * (p.penalty ? p.penalty[row0 + w] : 1.f)) : -INFINITY;
    p.parents[o] = w;
    p.tokens[o] = v;
    if (p.out_finished) p.out_finished[o] = !there || v == p.eos || m.ended[w];
  }
}

struct ScanPlan {
  int tiles;
  long long lists, tasks;
};
// As many segments as the GPU's SMs hold warps of the kernel, or fewer, where tiles are enough; more bins than candidates in each.  A row that
// does not begin on a 16-byte boundary may reach into one more tile.
static ScanPlan scan_plan(long long B, int W, long long V, int k, int ty, bool aligned) {
  const long long past = aligned ? 0 : 16 / elem_bytes(ty) - 1, row = (V + past + kTileLogits - 1) / kTileLogits;
  const long long held = 148 * kScanWarps * (ty == LETHE_F32 ? scan_ctas<LETHE_F32>(false) : scan_ctas<LETHE_BF16>(false));
  const long long want = (B * W * ((V + kTileLogits - 1) / kTileLogits) + held - 1) / held;
  ScanPlan s;
  s.tiles = static_cast<int>(want < kMostTiles ? want : kMostTiles);
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

template <int TY>
static int launch_beam(const BeamProblem& p, long long tasks, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>((tasks + kScanWarps - 1) / kScanWarps));
  if (p.allowed) beam_scan_kernel<TY, true><<<grid, 32 * kScanWarps, 0, st>>>(p);
  else beam_scan_kernel<TY, false><<<grid, 32 * kScanWarps, 0, st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return kErrLaunch;
  return launch_dependent(beam_merge_kernel<TY>, dim3(p.B), dim3(kMergeThreads), 0, st, p) == cudaSuccess ? kOk : kErrLaunch;
}

}  // namespace lg

extern "C" size_t lethe_gdn_beam_work_bytes(int64_t B, int32_t W, int64_t V, int32_t k, int32_t x_type) {
  using namespace lg;
  if (!beam_sizes(B, W, V, k, x_type)) return 0;
  return static_cast<size_t>(scan_plan(B, W, V, k, x_type, false).tasks) * (sizeof(ScanStat) + 8 * static_cast<size_t>(k + kSpare));
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
