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

#include "elem.cuh"
#include "host_util.h"
#include "umma.cuh"

namespace lg {

constexpr int kBeamMost = 64;                     // beams of a group, and candidates asked for
constexpr int kTileLogits = 1024, kMostTiles = 8; // a warp takes that many logits at a time, and so many times
constexpr int kScanWarps = 8, kFillWarps = 148 * 24;
constexpr int kCands = 256;                       // candidates of a segment that are put in order together
constexpr int kMergeThreads = 512, kBins = 128, kMergeRoom = 2 * kMergeThreads;
constexpr int kBehind = 8;                        // candidates behind the last chosen one that are looked at for equals
// A term of a sum: exp2 by the hardware 2^-22, its argument (two roundings of |t| 2^-24, weighted by 2^t) 2^-23.5, twice (tile to
// segment) the former, seven roundings of sums in 32 bits; the rest is in 64 bits.
constexpr double kLseError = 2 * 2.4e-7 + 1e-7 + 7 * 6e-8;

struct ScanStat {
  float m;          // largest logit
  int n;            // candidates in the list
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
  double temperature;
  ScanStat* stat;                         // [B, W, lists]
  unsigned long long* keys;               // [B, W, lists, k]
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
  // logits [v, v + N), minus infinity in the place of what is not there or not allowed; v + past is a multiple of N
  template <bool MASK> __device__ __forceinline__ Vec load(int v) const {
    Vec r;
    if (v >= 0 && v <= V - N) {
      r.load(x + v);
      if (MASK) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (!ok[v + i]) raw_put<TY, N>(r, i, least());
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) raw_put<TY, N>(r, i, at(v + i));
    }
    return r;
  }
};

// Segment of a row: the lanes' tiles lie 16 bytes a lane beside one another, so element e of vector n of a lane is token
// first + tile kTileLogits + n 32 N + lane N + e.
template <int TY, bool MASK>
__global__ void __launch_bounds__(32 * kScanWarps) beam_scan_kernel(const BeamProblem p) {
  using R = Row<TY>;
  __shared__ float2 bins[kScanWarps][kMostTiles][32];             // maximum and sum of a lane's part of a tile
  __shared__ unsigned long long cands[kScanWarps][kCands];
  __shared__ uint16_t passed[kScanWarps][kMostTiles * 32];
  griddep_launch();      // (the merge waits for the lists)
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long task = static_cast<long long>(blockIdx.x) * kScanWarps + warp;
  if (task >= static_cast<long long>(p.B) * p.W * p.lists) return;
  const int row = static_cast<int>(task / p.lists), seg = static_cast<int>(task % p.lists);
  if (!goes_on(p, row)) return;
  const R r(p, row);
  const int first = seg * p.tiles * kTileLogits - r.past;

  // sums and maxima
  float top = -INFINITY;
  for (int j = 0; j < p.tiles; ++j) {
    typename R::Vec x[R::kVecs];
#pragma unroll
    for (int n = 0; n < R::kVecs; ++n) x[n] = r.template load<MASK>(first + j * kTileLogits + (n * 32 + lane) * R::N);
    float m = -INFINITY;
#pragma unroll
    for (int n = 0; n < R::kVecs; ++n)
#pragma unroll
      for (int i = 0; i < R::N; ++i) m = fmaxf(m, x[n].get(i));
    const F2 less = f2(m == -INFINITY ? 0.f : -m), over = f2(p.over);
    F2 sum[4];
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      const F2 t = (x[n / (R::N / 2)].get2(n % (R::N / 2)) + less) * over;
      const F2 e = f2(ex2(lo(t)), ex2(hi(t)));
      sum[n % 4] = n < 4 ? e : sum[n % 4] + e;
    }
    const F2 s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    bins[warp][j][lane] = make_float2(m, lo(s) + hi(s));
    top = fmaxf(top, m);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
  double s = 0.;
  uint32_t best = 0, taken = 0;
  int best_at = 0;
  for (int j = 0; j < p.tiles; ++j) {
    const float2 bin = bins[warp][j][lane];
    s += static_cast<double>(bin.y * (bin.x == -INFINITY ? 0.f : ex2((bin.x - top) * p.over)));
    const uint32_t u = ordered(bin.x);
    if (u > best) best = u, best_at = j;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);

  // The k-th largest of the bins' maxima: what is below it is not among the k largest logits, and only bins that reach it have any of those.
  uint32_t least = 0;
  for (int i = 0; i < p.k; ++i) {
    least = __reduce_max_sync(~0u, best);
    if (least <= kLeast) break;
    if (lane == __ffs(__ballot_sync(~0u, best == least)) - 1) {
      taken |= 1u << best_at;
      best = 0;
      for (int j = 0; j < p.tiles; ++j) {
        const uint32_t u = (taken >> j) & 1u ? 0u : ordered(bins[warp][j][lane].x);
        if (u > best) best = u, best_at = j;
      }
    }
  }
  least = max(least, kLeast + 1);
  int reached = 0;
  for (int j = 0; j < p.tiles; ++j) {
    const bool mine = ordered(bins[warp][j][lane].x) >= least;
    const uint32_t who = __ballot_sync(~0u, mine);
    if (mine) passed[warp][reached + __popc(who & ((1u << lane) - 1))] = static_cast<uint16_t>(j * 32 + lane);
    reached += __popc(who);
  }
  __syncwarp();
  // their logits, one of a bin for each lane
  unsigned long long* const cand = cands[warp];
  int n = 0;
  constexpr int kAhead = 8;
  for (int i = 0; i < reached; i += kAhead) {
    uint32_t u[kAhead];
    int v[kAhead];
#pragma unroll
    for (int h = 0; h < kAhead; ++h) {
      const int bin = i + h < reached ? passed[warp][i + h] : 0;
      v[h] = first + bin / 32 * kTileLogits + (lane / R::N * 32 + bin % 32) * R::N + lane % R::N;
      u[h] = i + h < reached ? ordered(to_f32(r.at(v[h]))) : 0u;
    }
#pragma unroll
    for (int h = 0; h < kAhead; ++h) {
      const uint32_t who = __ballot_sync(~0u, u[h] >= least);
      const int at = n + __popc(who & ((1u << lane) - 1));
      if (u[h] >= least && at < kCands) cand[at] = static_cast<unsigned long long>(u[h]) << 32 | static_cast<uint32_t>(~v[h]);
      n += __popc(who);
    }
    if (n > kCands) break;
  }
  __syncwarp();
  unsigned long long* const list = p.keys + task * p.k;
  if (n <= kCands) {
    for (int i = lane; i < n; i += 32) {
      const unsigned long long key = cand[i];
      int before = 0;
      for (int j = 0; j < n; ++j) before += cand[j] > key;
      if (before < p.k) list[before] = key;
    }
    n = min(n, p.k);
  } else {
    // Too many equal ones, or large ones side by side: the largest of the segment, then the largest behind it, k times.
    unsigned long long last = ~0ull;
    for (n = 0; n < p.k; ++n) {
      unsigned long long key = 0;
      for (int j = 0; j < p.tiles * kTileLogits / 32; ++j) {
        const int v = first + j * 32 + lane;
        const uint32_t u = ordered(to_f32(r.at(v)));
        const unsigned long long c = static_cast<unsigned long long>(u) << 32 | static_cast<uint32_t>(~v);
        if (u > kLeast && c < last && c > key) key = c;
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) key = max(key, __shfl_xor_sync(~0u, key, d));
      if (!key) break;
      if (lane == 0) list[n] = key;
      last = key;
    }
  }
  if (lane == 0) p.stat[task] = ScanStat{top, n, s};
}

// A candidate: larger ones come first.
struct Entry {
  unsigned long long rank, place;      // ordered(r); ~(w V + v)
};
__device__ __forceinline__ bool larger(const Entry& a, const Entry& b) { return a.rank > b.rank || (a.rank == b.rank && a.place > b.place); }

struct MergeMemory {
  Entry room[kMergeRoom], sorted[kBins];
  double lse[kBeamMost], part[kMergeThreads / 32], widest;      // (largest 1 / penalty)
  float top[kBeamMost];
  bool on[kBeamMost], again[kBeamMost];
  int n, any;
};

// The largest of room[0, n), at most `most`, in order; `least` becomes the last of them where there are so many.
__device__ __forceinline__ void keep_largest(MergeMemory& m, int most, Entry* least) {
  __syncthreads();
  const int n = m.n;
  for (int i = threadIdx.x; i < n; i += kMergeThreads) {
    const Entry e = m.room[i];
    int before = 0;
    for (int j = 0; j < n; ++j) before += larger(m.room[j], e);
    if (before < most) m.sorted[before] = e;
  }
  __syncthreads();
  const int left = min(n, most);
  for (int i = threadIdx.x; i < left; i += kMergeThreads) m.room[i] = m.sorted[i];
  if (threadIdx.x == 0) m.n = left;
  if (left == most) *least = m.sorted[most - 1];
  __syncthreads();
}

template <int TY>
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamProblem p) {
  __shared__ MergeMemory m;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, row0 = blockIdx.x * p.W;
  const int lists = p.W * p.lists, most = p.k + kBehind;
  const ScanStat* const stat = p.stat + static_cast<long long>(row0) * p.lists;
  const unsigned long long* const keys = p.keys + static_cast<long long>(row0) * p.lists * p.k;
  griddep_wait();
  for (int w = warp; w < p.W; w += kMergeThreads / 32) {
    bool on = goes_on(p, row0 + w);
    float top = -INFINITY;
    double s = 0.;
    if (on) {
      const ScanStat* const a = stat + w * p.lists;
      for (int i = lane; i < p.lists; i += 32) top = fmaxf(top, a[i].m);
#pragma unroll
      for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
      for (int i = lane; i < p.lists; i += 32) {
        const ScanStat t = a[i];
        s += t.m == -INFINITY ? t.s : t.s * exp((static_cast<double>(t.m) - top) / p.temperature);
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
      on = s > 0. && s < INFINITY && top < INFINITY;
    }
    if (lane == 0) {
      m.on[w] = on;
      m.top[w] = top;
      m.lse[w] = on ? top / p.temperature + log(s) : 0.;
      m.again[w] = false;
    }
  }
  auto penalty = [&](int w) { return p.penalty ? static_cast<double>(p.penalty[row0 + w]) : 1.; };
  auto entry = [&](int l, unsigned long long key) {
    const int w = l / p.lists;
    const double x = static_cast<double>(from_ordered(static_cast<uint32_t>(key >> 32))) / p.temperature;
    const double c = static_cast<double>(p.scores[row0 + w]) + (x - m.lse[w]);
    return Entry{ordered(c / penalty(w)), ~(static_cast<unsigned long long>(w) * p.V + static_cast<uint32_t>(~static_cast<uint32_t>(key)))};
  };
  for (int pass = 0;; ++pass) {
    __syncthreads();
    if (tid == 0) {
      m.n = m.any = 0;
      m.widest = 0.;
      for (int w = 0; w < p.W; ++w)
        if (counts(p, row0 + w)) m.widest = fmax(m.widest, 1. / penalty(w));
    }
    __syncthreads();
    if (tid < p.W && p.finished && p.finished[row0 + tid] && counts(p, row0 + tid))
      m.room[atomicAdd(&m.n, 1)] = Entry{ordered(p.scores[row0 + tid] / penalty(tid)), ~(static_cast<unsigned long long>(tid) * p.V + p.eos)};
    // The `most`-th largest of the bins' first candidates, of which none of those behind it is among the `most` largest.
    Entry least{0, 0}, head{0, 0};
    for (int l = tid; l < lists; l += kMergeThreads)
      if (m.on[l / p.lists] && stat[l].n > 0) {
        const Entry e = entry(l, keys[static_cast<long long>(l) * p.k]);
        if (larger(e, head)) head = e;
      }
#pragma unroll
    for (int d = kMergeThreads / kBins / 2; d; d >>= 1) {
      const Entry e{__shfl_xor_sync(~0u, head.rank, d), __shfl_xor_sync(~0u, head.place, d)};
      if (larger(e, head)) head = e;
    }
    if (tid % (kMergeThreads / kBins) == 0) m.sorted[tid / (kMergeThreads / kBins)] = head;
    __syncthreads();
    if (tid < kBins) {
      const Entry e = m.sorted[tid];
      int before = 0;
      for (int j = 0; j < kBins; ++j) before += larger(m.sorted[j], e);
      if (before == most - 1 && e.rank) m.room[kMergeRoom - 1] = e, m.any = 1;
    }
    __syncthreads();
    if (m.any) least = m.room[kMergeRoom - 1];
    __syncthreads();
    // every thread's lists, each to its first candidate below `least`
    int l = tid, at = 0;
    for (;;) {
      Entry e{0, 0};
      bool have = false;
      while (l < lists && !have) {
        if (m.on[l / p.lists] && at < stat[l].n) {
          e = entry(l, keys[static_cast<long long>(l) * p.k + at]);
          have = !larger(least, e);
        }
        if (!have) l += kMergeThreads, at = 0;
      }
      if (have) {
        m.room[atomicAdd(&m.n, 1)] = e;
        ++at;
      }
      if (!__syncthreads_or(have)) break;
      const int n = m.n;
      __syncthreads();
      if (n > kMergeRoom - kMergeThreads) keep_largest(m, most, &least);
    }
    keep_largest(m, most, &least);
    if (pass) break;
    // Candidates of different beams next to one another, closer than the sums are known.
    if (tid == 0) m.any = 0;
    __syncthreads();
    const int n = m.n;
    auto beam = [&](const Entry& e) { return static_cast<int>(~e.place / p.V); };
    auto doubt = [&](const Entry& a, const Entry& b) {
      const int u = beam(a), w = beam(b);
      const double gap = from_ordered(a.rank) - from_ordered(b.rank);
      return gap > 0. && u != w && gap < kLseError * (1. / penalty(u) + 1. / penalty(w));
    };
    if (tid < n && tid < p.k) {
      const Entry a = m.sorted[tid];
      const double far = 2. * kLseError * m.widest;
      int j = tid + 1;
      for (; j < n && from_ordered(a.rank) - from_ordered(m.sorted[j].rank) < far; ++j)
        if (doubt(a, m.sorted[j])) m.again[beam(a)] = m.again[beam(m.sorted[j])] = m.any = 1;
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
      for (int v = tid; v < p.V; v += kMergeThreads)
        s += exp((static_cast<double>(to_f32(r.at(v))) - m.top[w]) / p.temperature);
#pragma unroll
      for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
      if (lane == 0) m.part[warp] = s;
      __syncthreads();
      if (tid == 0) {
        s = 0.;
        for (int i = 0; i < kMergeThreads / 32; ++i) s += m.part[i];
        m.lse[w] = m.top[w] / p.temperature + log(s);
      }
      __syncthreads();
    }
  }
  if (tid < p.k) {
    const long long o = static_cast<long long>(blockIdx.x) * p.k + tid;
    const bool there = tid < m.n;
    const unsigned long long place = there ? ~m.sorted[tid].place : 0;
    const int w = static_cast<int>(place / p.V), v = there ? static_cast<int>(place % p.V) : max(p.eos, 0);
    p.out_scores[o] = there ? static_cast<float>(from_ordered(m.sorted[tid].rank) * penalty(w)) : -INFINITY;
    p.parents[o] = w;
    p.tokens[o] = v;
    if (p.out_finished) p.out_finished[o] = !there || v == p.eos || (p.finished && p.finished[row0 + w]);
  }
}

struct ScanPlan {
  int tiles;
  long long lists, tasks;
};
// Segments short enough for kFillWarps of them, where there are so many; more bins than candidates in each.
static ScanPlan scan_plan(long long B, int W, long long V, int k, int ty) {
  const long long n = 16 / elem_bytes(ty), row = (V + n - 1 + kTileLogits - 1) / kTileLogits;
  ScanPlan s;
  const long long want = B * W * row / kFillWarps;
  s.tiles = static_cast<int>(want < kMostTiles ? want : kMostTiles);
  if (s.tiles * 32 < k) s.tiles = (k + 31) / 32;
  s.lists = (row + s.tiles - 1) / s.tiles;
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
  return static_cast<size_t>(scan_plan(B, W, V, k, x_type).tasks) * (sizeof(ScanStat) + 8 * static_cast<size_t>(k));
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
  const ScanPlan plan = scan_plan(a->B, a->W, a->V, a->k, a->x_type);
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
  p.temperature = a->temperature;
  p.over = static_cast<float>(1.4426950408889634 / p.temperature);
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
