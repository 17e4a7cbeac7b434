// The states of sequences as rows of tensors: every beam takes over its parent's row (reorder), sequences get free rows and a copy of
// another's (fork), the rows in use move together (compact).  Nothing is computed: what bounds these is reading every row
// that somebody takes over once and writing every row that changes once.  Which rows those are stands on the device; every CTA works it
// out for itself (bytes against megabytes) instead of waiting for a launch that does.
#include "elem.cuh"
#include "host_util.h"
#include "umma.cuh"

namespace lg {

constexpr int kRowThreads = 256, kRowCtas = 4;
constexpr int kMostTensors = 32;            // of one launch
constexpr int kMostBeams = 256, kMostSlots = 65536, kMostEntries = 4096;
constexpr int kReorderBytes = 32768, kCopyStrip = 16384;

struct StateTensor {
  char* data;
  long long row, stride, group;     // bytes
  int unit, strip;                  // what is moved at once; bytes of a row that a CTA takes
  long long first;                  // places of the tensors in front
};
struct StateTensors {
  StateTensor t[kMostTensors];
  int count;
};

__device__ __forceinline__ const StateTensor& tensor_of(const StateTensors& s, long long item) {
  int i = 0;
  while (i + 1 < s.count && item >= s.t[i + 1].first) ++i;
  return s.t[i];
}

template <int U> struct Unit;
template <> struct Unit<16> { using T = uint4; };
template <> struct Unit<8> { using T = uint2; };
template <> struct Unit<4> { using T = uint32_t; };
template <> struct Unit<2> { using T = uint16_t; };
template <> struct Unit<1> { using T = uint8_t; };

template <typename F> __device__ __forceinline__ void with_unit(int unit, F&& f) {
  switch (unit) {
    case 16: f(Unit<16>()); break;
    case 8: f(Unit<8>()); break;
    case 4: f(Unit<4>()); break;
    case 2: f(Unit<2>()); break;
    default: f(Unit<1>()); break;
  }
}

// Sum over the threads in front, and over all.
__device__ __forceinline__ unsigned block_scan(unsigned x, unsigned* total) {
  __shared__ unsigned warps[kRowThreads / 32];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  unsigned s = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const unsigned y = __shfl_up_sync(~0u, s, d);
    if (lane >= d) s += y;
  }
  __syncthreads();
  if (lane == 31) warps[warp] = s;
  __syncthreads();
  unsigned before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kRowThreads / 32; ++w) {
    if (w < warp) before += warps[w];
    all += warps[w];
  }
  *total = all;
  return before + s - x;
}

__device__ __forceinline__ long long index_at(const void* p, int is64, long long i) {
  return is64 ? static_cast<const long long*>(p)[i] : static_cast<const int*>(p)[i];
}

// ------------------------------------------------------------------------------------------------------------------
// Reorder: a CTA has a strip of the rows of one group.  The strips that somebody takes over are in shared memory before any is written.
// ------------------------------------------------------------------------------------------------------------------
struct ReorderProblem {
  StateTensors s;
  const void* parents;
  int parents64, W;
  int* status;
};

template <typename T> __device__ __forceinline__ void fetch(T* to, const T* from) {
  if constexpr (sizeof(T) >= 4) {
    const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(to));
    if constexpr (sizeof(T) == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(from), "n"(sizeof(T)) : "memory");
  } else {
    *to = *from;
  }
}

__global__ void __launch_bounds__(kRowThreads) reorder_kernel(const __grid_constant__ ReorderProblem p) {
  extern __shared__ __align__(16) char strips[];
  __shared__ int used[kMostBeams], sources[kMostBeams], to[kMostBeams], from[kMostBeams];
  const int tid = threadIdx.x;
  const StateTensor& t = tensor_of(p.s, blockIdx.x);
  const long long item = blockIdx.x - t.first, per = (t.row + t.strip - 1) / t.strip;
  const long long b = item / per, begin = item % per * t.strip;
  const int width = static_cast<int>(min(static_cast<long long>(t.strip), t.row - begin));

  long long parent = tid < p.W ? index_at(p.parents, p.parents64, b * p.W + tid) : tid;
  if (parent < 0 || (tid < p.W && parent >= p.W)) {
    *p.status = kErrIndex;
    parent = tid;
  }
  used[tid] = 0;
  __syncthreads();
  const bool moves = tid < p.W && parent != tid;
  if (moves) used[parent] = 1;
  __syncthreads();
  const bool source = used[tid];
  unsigned both;
  const unsigned at = block_scan(moves | source << 16, &both);
  if (source) {
    sources[at >> 16] = tid;
    used[tid] = at >> 16;
  }
  __syncthreads();
  if (moves) {
    to[at & 0xffff] = tid;
    from[at & 0xffff] = used[parent];
  }
  const int n = both & 0xffff, reads = static_cast<int>(both >> 16);
  char* const rows = t.data + b * t.group + begin;
  with_unit(t.unit, [&](auto u) {
    using T = typename decltype(u)::T;
    const int columns = width / static_cast<int>(sizeof(T));
    T* const mine = reinterpret_cast<T*>(strips);
    for (int i = tid; i < reads * columns; i += kRowThreads)
      fetch(mine + i, reinterpret_cast<const T*>(rows + sources[i / columns] * t.stride) + i % columns);
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    for (int i = tid; i < n * columns; i += kRowThreads)
      reinterpret_cast<T*>(rows + to[i / columns] * t.stride)[i % columns] = mine[from[i / columns] * columns + i % columns];
  });
}

// ------------------------------------------------------------------------------------------------------------------
// Fork and compact: a list of rows that are read and rows that are written, none of them both
// ------------------------------------------------------------------------------------------------------------------
struct PoolProblem {
  StateTensors s;
  long long strips;                 // of all tensors' rows
  const uint8_t* live;
  int slots;
  // fork
  const void* source;
  int source64, n;
  long long* target;
  uint8_t* after;
  // compact
  long long *place, *live_count;
};

// Strip after strip of every move: the rows that share a source read the same strip of it at about the same time, from L2 all but once.
template <typename Src, typename Dst>
__device__ __forceinline__ void copy_rows(const PoolProblem& p, int moves, Src src, Dst dst) {
  for (long long item = blockIdx.x; item < p.strips * moves; item += gridDim.x) {
    const long long strip = item / moves;
    const int m = static_cast<int>(item % moves);
    const StateTensor& t = tensor_of(p.s, strip);
    const long long begin = (strip - t.first) * t.strip;
    const int width = static_cast<int>(min(static_cast<long long>(t.strip), t.row - begin));
    const long long s = src(m);
    with_unit(t.unit, [&](auto u) {
      using T = typename decltype(u)::T;
      constexpr int kAhead = 4;
      const int columns = width / static_cast<int>(sizeof(T));
      const T* const in = reinterpret_cast<const T*>(t.data + s * t.stride + begin);
      T* const out = reinterpret_cast<T*>(t.data + dst(m) * t.stride + begin);
      for (int c = threadIdx.x; c < columns; c += kAhead * kRowThreads) {
        T x[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          x[i] = T{};
          if (s >= 0 && c + i * kRowThreads < columns) x[i] = in[c + i * kRowThreads];
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
          if (c + i * kRowThreads < columns) out[c + i * kRowThreads] = x[i];
      }
    });
  }
}

__global__ void __launch_bounds__(kRowThreads, kRowCtas) fork_kernel(const __grid_constant__ PoolProblem p) {
  extern __shared__ int lists[];
  int *const slot = lists, *const src = lists + p.n;
  const int tid = threadIdx.x;
  // the lowest n free slots
  const int each = (p.slots + kRowThreads - 1) / kRowThreads, s0 = min(p.slots, tid * each), s1 = min(p.slots, s0 + each);
  int free = 0;
  for (int s = s0; s < s1; ++s) free += !p.live[s];
  unsigned frees, total;
  const int before = block_scan(free, &frees);
  int at = before;
  for (int s = s0; s < s1 && at < p.n; ++s)
    if (!p.live[s]) slot[at++] = s;
  __syncthreads();
  // the entries that take one
  const int per = (p.n + kRowThreads - 1) / kRowThreads, e0 = min(p.n, tid * per), e1 = min(p.n, e0 + per);
  auto takes = [&](int e) {
    const long long s = index_at(p.source, p.source64, e);
    return s == -1 || (s >= 0 && s < p.slots && p.live[s]);
  };
  int mine = 0;
  for (int e = e0; e < e1; ++e) mine += takes(e);
  at = block_scan(mine, &total);
  const int moves = min(total, frees);
  for (int e = e0; e < e1; ++e) {
    long long got = -1;
    if (takes(e)) {
      if (at < moves) {
        got = slot[at];
        src[at] = static_cast<int>(index_at(p.source, p.source64, e));
      }
      ++at;
    }
    if (blockIdx.x == 0) p.target[e] = got;
  }
  if (blockIdx.x == 0) {
    at = before;
    for (int s = s0; s < s1; ++s) p.after[s] = p.live[s] || at++ < moves;
  }
  __syncthreads();
  copy_rows(p, moves, [&](int m) { return static_cast<long long>(src[m]); }, [&](int m) { return static_cast<long long>(slot[m]); });
}

__global__ void __launch_bounds__(kRowThreads, kRowCtas) compact_kernel(const __grid_constant__ PoolProblem p) {
  extern __shared__ uint16_t rows[];
  uint16_t *const src = rows, *const dst = rows + p.slots / 2;
  const int tid = threadIdx.x;
  const int each = (p.slots + kRowThreads - 1) / kRowThreads, s0 = min(p.slots, tid * each), s1 = min(p.slots, s0 + each);
  unsigned live = 0, total;
  for (int s = s0; s < s1; ++s) live += p.live[s] != 0;
  block_scan(live, &total);
  const int count = total;
  // those behind the place of the last live slot to be, and the holes in front of it: as many of one as of the other
  unsigned both = 0;
  for (int s = s0; s < s1; ++s) both += p.live[s] ? s >= count : (s < count ? 1u << 16 : 0u);
  const unsigned before = block_scan(both, &total);
  const int moves = total & 0xffff;
  int leave = before & 0xffff, hole = before >> 16;
  for (int s = s0; s < s1; ++s) {
    if (p.live[s]) {
      if (s >= count) src[leave++] = static_cast<uint16_t>(s);
    } else if (s < count) {
      dst[hole++] = static_cast<uint16_t>(s);
    }
  }
  __syncthreads();
  leave = before & 0xffff;
  for (int s = s0; s < s1; ++s) {
    long long to = -1;
    if (p.live[s]) to = s < count ? s : dst[leave++];
    if (static_cast<unsigned>(s) % gridDim.x == blockIdx.x) p.place[s] = to;
  }
  if (blockIdx.x == 0 && tid == 0) *p.live_count = count;
  copy_rows(p, moves, [&](int m) { return static_cast<long long>(src[m]); }, [&](int m) { return static_cast<long long>(dst[m]); });
}

// ------------------------------------------------------------------------------------------------------------------
// The tensors [begin, ...) of a call that go into one launch; `groups`: how often each is counted.  Returns an error code.
static int take_states(const LetheGdnStates* s, int count, int strip, long long groups, StateTensors* out, long long* items) {
  long long n = 0;
  out->count = count;
  for (int i = 0; i < count; ++i) {
    StateTensor& t = out->t[i];
    t.data = static_cast<char*>(s[i].data);
    t.row = s[i].row_bytes;
    t.stride = s[i].stride;
    t.group = s[i].group_stride;
    const unsigned long long bits = reinterpret_cast<uintptr_t>(t.data) | t.row | t.stride | t.group;
    t.unit = 16;
    while (bits % t.unit) t.unit /= 2;
    t.strip = strip;
    t.first = n;
    n += groups * ((t.row + strip - 1) / strip);
  }
  *items = n;
  return kOk;
}
static int check_states(const LetheGdnStates* s, int count) {
  if (count < 0 || (count && !s)) return kErrNull;
  for (int i = 0; i < count; ++i) {
    if (!s[i].data) return kErrNull;
    if (s[i].row_bytes <= 0 || s[i].row_bytes > (1ll << 40)) return kErrDims;
  }
  return kOk;
}

template <typename Launch>
static int in_launches(const LetheGdnStates* states, int count, int strip, long long groups, Launch launch) {
  for (int i = 0; i == 0 || i < count; i += kMostTensors) {
    StateTensors s;
    long long items;
    take_states(states + i, count - i < kMostTensors ? count - i : kMostTensors, strip, groups, &s, &items);
    const int rc = launch(s, items);
    if (rc != kOk) return rc;
  }
  return kOk;
}

}  // namespace lg

extern "C" int lethe_gdn_reorder_states(const LetheGdnStates* states, int32_t count, int64_t B, int32_t W, const void* parents, int32_t parents_64,
                                        int32_t* status, void* stream) {
  using namespace lg;
  if (!parents || !status || count < 1) return kErrNull;
  const int bad = check_states(states, count);
  if (bad) return bad;
  if (B <= 0 || W <= 0 || W > kMostBeams || B > (1ll << 30)) return kErrDims;
  if (reinterpret_cast<uintptr_t>(parents) % (parents_64 ? 8 : 4)) return kErrAlign;
  int strip = 128;
  while (strip < kCopyStrip && 2 * strip * W <= kReorderBytes) strip *= 2;
  for (int i = 0; i < count; ++i)
    if ((states[i].row_bytes + strip - 1) / strip > (1ll << 30) / kMostTensors / B) return kErrDims;
  DeviceGuard guard(states[0].data);
  if (!guard.ok) return kErrDevice;
  return in_launches(states, count, strip, B, [&](const StateTensors& s, long long items) {
    ReorderProblem p;
    p.s = s;
    p.parents = parents;
    p.parents64 = parents_64;
    p.W = W;
    p.status = status;
    reorder_kernel<<<static_cast<unsigned>(items), kRowThreads, kReorderBytes, static_cast<cudaStream_t>(stream)>>>(p);
    return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
  });
}

static int pool_call(const LetheGdnStates* states, int count, long long slots, const uint8_t* live, lg::PoolProblem* p, bool fork, size_t smem,
                     long long most, void* stream) {
  using namespace lg;
  DeviceGuard guard(live);
  if (!guard.ok) return kErrDevice;
  const int sms = sm_count();
  if (sms <= 0) return kErrDevice;
  static SmemAttr attrs[2];
  if (attrs[fork].set(fork ? fork_kernel : compact_kernel, fork ? 8 * kMostEntries : 2 * kMostSlots)) return kErrLaunch;
  p->live = live;
  p->slots = static_cast<int>(slots);
  return in_launches(states, count, kCopyStrip, 1, [&](const StateTensors& s, long long strips) {
    p->s = s;
    p->strips = strips;
    const long long items = strips * most, ctas = static_cast<long long>(kRowCtas) * sms;
    const unsigned grid = static_cast<unsigned>(items < 1 ? 1 : items < ctas ? items : ctas);
    (fork ? fork_kernel : compact_kernel)<<<grid, kRowThreads, smem, static_cast<cudaStream_t>(stream)>>>(*p);
    return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
  });
}

extern "C" int lethe_gdn_fork_states(const LetheGdnStates* states, int32_t count, int64_t slots, const uint8_t* live, const void* source,
                                     int32_t source_64, int64_t n, int64_t* target, uint8_t* live_after, void* stream) {
  using namespace lg;
  if (!live || !source || !target || !live_after) return kErrNull;
  const int bad = check_states(states, count);
  if (bad) return bad;
  if (slots <= 0 || slots > kMostSlots || n <= 0 || n > kMostEntries) return kErrDims;
  if (reinterpret_cast<uintptr_t>(source) % (source_64 ? 8 : 4) || reinterpret_cast<uintptr_t>(target) % 8) return kErrAlign;
  PoolProblem p = {};
  p.source = source;
  p.source64 = source_64;
  p.n = static_cast<int>(n);
  p.target = reinterpret_cast<long long*>(target);
  p.after = live_after;
  return pool_call(states, count, slots, live, &p, true, 8 * static_cast<size_t>(n), n < slots ? n : slots, stream);
}

extern "C" int lethe_gdn_compact_states(const LetheGdnStates* states, int32_t count, int64_t slots, const uint8_t* live, int64_t* place,
                                        int64_t* live_count, void* stream) {
  using namespace lg;
  if (!live || !place || !live_count) return kErrNull;
  const int bad = check_states(states, count);
  if (bad) return bad;
  if (slots <= 0 || slots > kMostSlots) return kErrDims;
  if ((reinterpret_cast<uintptr_t>(place) | reinterpret_cast<uintptr_t>(live_count)) % 8) return kErrAlign;
  PoolProblem p = {};
  p.place = reinterpret_cast<long long*>(place);
  p.live_count = reinterpret_cast<long long*>(live_count);
  return pool_call(states, count, slots, live, &p, false, 2 * static_cast<size_t>(slots), slots / 2, stream);
}
