// The states of sequences as rows of tensors: every beam takes over its parent's row (reorder), sequences get free rows and a copy of
// another's (fork), the rows in use move together (compact).  Nothing is computed: what bounds these is reading every row
// that somebody takes over once and writing every row that changes once.  Which rows those are stands on the device; every CTA works it
// out for itself (bytes against megabytes) instead of waiting for a launch that does.
//
// Measured, a pass through the public call: reorder of 64 x 8 rows of 2 MB, 6 moved from 3 in each group (1.23 GB, 187 us at the copy rate) 218 us; 272 rows of
// 2 MB forked from 32 and from zeros (0.65 GB, 98 us) 125 us; 128 rows moved (0.54 GB, 83 us) 93 us; a few small rows 5 to 7 us, which is
// the host's time.  HBM moves what the rows have and no more (409 MB in and 757 out, 80 and 514, 272 and 218); two writes for a read run at 5.6 TB/s.
//
// Rows of 16-byte multiples go through shared memory by bulk copies, one CTA per SM: up to four warps issue them, each with a ring of its own,
// and no thread touches the data.  Rows of other sizes go through registers in the other warps meanwhile.
#include "elem.cuh"
#include "host_util.h"
#include "state_ring.cuh"

namespace lg {

constexpr int kRowThreads = 256, kPlainWarps = kRowThreads / 32 - kCopyWarps;
constexpr int kMostTensors = 32;            // of one launch
constexpr int kMostBeams = 256, kMostSlots = 65536, kMostEntries = 4096;
constexpr int kGroupBytes = 32768;          // a wide group's strips
constexpr int kAllBytes = 208896, kMostStage = 8192;      // dynamic shared memory of a CTA; bytes of a stage where there are four rings
constexpr int kSiteReorder = 811, kSiteCopy = 812;

struct StateTensor {
  char* data;
  long long row, stride, group;     // bytes
  int unit, strip;                  // what is moved at once; bytes of a row that are an item's
  long long first;                  // strips of the tensors in front
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

template <typename T> __device__ __forceinline__ void fetch(T* to, const T* from) {
  if constexpr (sizeof(T) == 4 || sizeof(T) == 8) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(to)), "l"(from), "n"(sizeof(T)) : "memory");
  } else if constexpr (sizeof(T) == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(from) : "memory");
  } else {
    *to = *from;
  }
}

// a / b, and what is left
__device__ __forceinline__ unsigned long long divide(unsigned long long a, unsigned b, unsigned* rest) {
  const unsigned long long q = a >> 32 ? a / b : static_cast<unsigned>(a) / b;
  *rest = static_cast<unsigned>(a - q * b);
  return q;
}

__device__ __forceinline__ long long index_at(const void* p, int is64, long long i) {
  return is64 ? static_cast<const long long*>(p)[i] : static_cast<const int*>(p)[i];
}

// the copying warps' items: first those of one warp of every CTA
__device__ __forceinline__ long long first_item() { return static_cast<long long>(threadIdx.x / 32) * gridDim.x + blockIdx.x; }

// ------------------------------------------------------------------------------------------------------------------
// Reorder.  An item is a strip of the rows of one group, a step as much of it as a stage holds: those that somebody takes over are in
// shared memory before any is written.
// ------------------------------------------------------------------------------------------------------------------
struct ReorderProblem {
  StateTensors bulk, plain;
  long long bulk_items, plain_items;
  const void* parents;
  int parents64, W, copy_warps, stage_bytes;
  int* status;
};

struct Parents {              // of a group of up to 32, in a warp's lanes
  int parent;
  uint32_t used;              // rows that others take over
  bool moves;
  __device__ __forceinline__ int place(int row) const { return __popc(used & ((1u << row) - 1)); }
};
__device__ __forceinline__ long long parent_of(const ReorderProblem& p, long long b) {
  const int lane = threadIdx.x % 32;
  return lane < p.W ? index_at(p.parents, p.parents64, b * p.W + lane) : lane;
}
__device__ __forceinline__ Parents parents_of(const ReorderProblem& p, long long x) {
  const int lane = threadIdx.x % 32;
  if (x < 0 || (lane < p.W && x >= p.W)) {
    report(p.status, kErrIndex);
    x = lane;
  }
  Parents r;
  r.parent = static_cast<int>(x);
  r.moves = r.parent != lane;
  r.used = __reduce_or_sync(~0u, r.moves ? 1u << r.parent : 0u);
  return r;
}

struct Strip {
  const StateTensor* t;
  long long group, begin;
  int width;
};
__device__ __forceinline__ Strip strip_of(const StateTensors& s, long long item) {
  const StateTensor& t = tensor_of(s, item);
  unsigned rest;
  Strip r;
  r.t = &t;
  r.group = divide(item - t.first, static_cast<unsigned>((t.row + t.strip - 1) / t.strip), &rest);
  r.begin = static_cast<long long>(rest) * t.strip;
  r.width = static_cast<int>(min(static_cast<long long>(t.strip), t.row - r.begin));
  return r;
}

__global__ void __launch_bounds__(kRowThreads) reorder_kernel(const __grid_constant__ ReorderProblem p) {
  extern __shared__ __align__(128) unsigned char memory[];
  __shared__ RingMemory rings;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  Ring ring(rings, memory, p.stage_bytes, p.status, kSiteReorder);
  __syncthreads();
  griddep_wait();
  if (warp < p.copy_warps) {
    long long item = first_item(), ahead = 0;      // ahead: the lane's parent in the next item
    const long long step = static_cast<long long>(p.copy_warps) * gridDim.x;
    if (item < p.bulk_items) ahead = parent_of(p, strip_of(p.bulk, item).group);
    Strip x;
    Parents r;
    int done = 0, width = 0;
    x.width = 0;
    ring.run([&](int s, LaneCopy* c) {
      while (done >= x.width) {
        if (item >= p.bulk_items) return false;
        x = strip_of(p.bulk, item);
        r = parents_of(p, ahead);
        item += step;
        if (item < p.bulk_items) ahead = parent_of(p, strip_of(p.bulk, item).group);
        const int reads = __popc(r.used);
        done = reads ? 0 : x.width;
        width = reads ? ring.stage_bytes / reads / 128 * 128 : 0;
      }
      const int n = min(width, x.width - done);
      char* const row = x.t->data + x.group * x.t->group + lane * x.t->stride + x.begin + done;
      ring.expect(s, __popc(r.used) * n);
      if ((r.used >> lane) & 1) bulk_g2s(ring.stage(s) + r.place(lane) * width, row, n, ring.full + s);
      *c = LaneCopy{row, smem_u32(ring.stage(s) + r.place(r.parent) * width), r.moves ? static_cast<uint32_t>(n) : 0u};
      done += n;
      return true;
    });
    return;
  }
  if (warp < kCopyWarps) return;
  // The others: a column of units for each lane, which has all rows of it in its own places of shared memory before it writes one.
  unsigned char* const own = memory + kStages * p.copy_warps * p.stage_bytes + (warp - kCopyWarps) * p.W * 32 * 8;
  for (long long item = static_cast<long long>(blockIdx.x) * kPlainWarps + warp - kCopyWarps; item < p.plain_items; item += static_cast<long long>(gridDim.x) * kPlainWarps) {
    const Strip x = strip_of(p.plain, item);
    const Parents r = parents_of(p, parent_of(p, x.group));
    const uint32_t moved = __ballot_sync(~0u, r.moves);
    char* const rows = x.t->data + x.group * x.t->group + x.begin;
    with_unit(x.t->unit, [&](auto u) {
      using T = typename decltype(u)::T;
      T* const mine = reinterpret_cast<T*>(own) + lane;
      for (int c = lane; c < (x.width / static_cast<int>(sizeof(T)) + 31) / 32 * 32; c += 32) {
        const bool in = c < x.width / static_cast<int>(sizeof(T));
        int n = 0;
        for (uint32_t m = r.used; m; m &= m - 1, ++n)
          if (in) fetch(mine + n * 32, reinterpret_cast<const T*>(rows + (__ffs(m) - 1) * x.t->stride) + c);
        asm volatile("cp.async.wait_all;" ::: "memory");
        for (uint32_t m = moved; m; m &= m - 1) {
          const int row = __ffs(m) - 1, from = r.place(__shfl_sync(~0u, r.parent, row));
          if (in) reinterpret_cast<T*>(rows + row * x.t->stride)[c] = mine[from * 32];
        }
      }
    });
  }
}

// Groups of more than 32 rows: an item at a time for each CTA, all of its threads.
constexpr long long kMostWideCtas = 65536;
__global__ void __launch_bounds__(kRowThreads) reorder_wide_kernel(const __grid_constant__ ReorderProblem p) {
  extern __shared__ __align__(128) unsigned char memory[];
  __shared__ int used[kMostBeams], sources[kMostBeams], to[kMostBeams], from[kMostBeams];
  const int tid = threadIdx.x;
  griddep_wait();
  for (long long item = blockIdx.x; item < p.plain_items; item += gridDim.x) {
    const Strip x = strip_of(p.plain, item);
    long long parent = tid < p.W ? index_at(p.parents, p.parents64, x.group * p.W + tid) : tid;
    if (parent < 0 || (tid < p.W && parent >= p.W)) {
      report(p.status, kErrIndex);
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
    char* const rows = x.t->data + x.group * x.t->group + x.begin;
    with_unit(x.t->unit, [&](auto u) {
      using T = typename decltype(u)::T;
      const int columns = x.width / static_cast<int>(sizeof(T));
      T* const mine = reinterpret_cast<T*>(memory);
      for (int i = tid; i < reads * columns; i += kRowThreads)
        fetch(mine + i, reinterpret_cast<const T*>(rows + sources[i / columns] * x.t->stride) + i % columns);
      asm volatile("cp.async.wait_all;" ::: "memory");
      __syncthreads();
      for (int i = tid; i < n * columns; i += kRowThreads)
        reinterpret_cast<T*>(rows + to[i / columns] * x.t->stride)[i % columns] = mine[from[i / columns] * columns + i % columns];
    });
    __syncthreads();      // (the next item's lists and columns go where these are)
  }
}

// ------------------------------------------------------------------------------------------------------------------
// Fork and compact: a list of rows that are read and rows that are written, none of them both
// ------------------------------------------------------------------------------------------------------------------
constexpr int kGroupSlots = 4096, kGroupEntries = 1024, kMostTargets = 8;      // moves are put together by their source up to here; of one load
constexpr double kTogetherBytes = 32e6;      // (272 rows of 2 MB: 140 us one by one, 125 together)

struct PoolProblem {
  StateTensors bulk, plain;
  long long bulk_strips, plain_strips;      // of all tensors' rows
  const uint8_t* live;
  int slots, stage_bytes;               // (a strip of a bulk row is a stage)
  int* status;
  // fork
  const void* source;
  int source64, n, together;            // together: moves of one source share its loads
  long long* target;
  uint8_t* after;
  // compact
  long long *place, *live_count;
};
// shared memory: the ring, a strip of zeros (fork), lists
constexpr int fork_list_bytes(int slots, int n, bool together) { return 8 * n + (together ? 4 * (slots + 2) + 14 * n + 8 : 0); }

// `chunks` of moves: row src(i) goes to rows dst(i, 0 ... len(i) - 1); `moves` single ones for rows that are not of 16-byte multiples.
// The strips of a chunk one after another, so that the CTAs are near one another in memory.
template <typename Src, typename Len, typename Dst, typename From, typename To>
__device__ __forceinline__ void copy_rows(const PoolProblem& p, Ring& ring, const unsigned char* zeros, int chunks, Src src, Len len, Dst dst, int moves, From from, To to) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  auto strip = [](const StateTensors& s, long long i) {
    const StateTensor& t = tensor_of(s, i);
    const long long begin = (i - t.first) * t.strip;
    return Strip{&t, 0, begin, static_cast<int>(min(static_cast<long long>(t.strip), t.row - begin))};
  };
  if (warp < kCopyWarps) {
    long long item = first_item();
    ring.run([&](int s, LaneCopy* out) {
      if (item >= p.bulk_strips * chunks) return false;
      unsigned i;
      const int c = static_cast<int>(divide(item, static_cast<unsigned>(p.bulk_strips), &i));
      const Strip x = strip(p.bulk, i);
      item += kCopyWarps * gridDim.x;
      const long long row = src(c);
      if (row >= 0) {
        ring.expect(s, x.width);
        if (lane == 0) bulk_g2s(ring.stage(s), x.t->data + row * x.t->stride + x.begin, x.width, ring.full + s);
      }
      *out = LaneCopy{nullptr, 0, 0};
      if (lane < len(c)) *out = LaneCopy{x.t->data + static_cast<long long>(dst(c, lane)) * x.t->stride + x.begin, smem_u32(row < 0 ? zeros : ring.stage(s)), static_cast<uint32_t>(x.width)};
      return true;
    });
    return;
  }
  for (long long item = static_cast<long long>(blockIdx.x) * kPlainWarps + warp - kCopyWarps; item < p.plain_strips * moves; item += static_cast<long long>(gridDim.x) * kPlainWarps) {
    unsigned i;
    const int m = static_cast<int>(divide(item, static_cast<unsigned>(p.plain_strips), &i));
    const Strip x = strip(p.plain, i);
    const long long row = from(m);
    with_unit(x.t->unit, [&](auto u) {
      using T = typename decltype(u)::T;
      constexpr int kAhead = 8;
      const int columns = x.width / static_cast<int>(sizeof(T));
      const T* const in = reinterpret_cast<const T*>(x.t->data + row * x.t->stride + x.begin);
      T* const out = reinterpret_cast<T*>(x.t->data + static_cast<long long>(to(m)) * x.t->stride + x.begin);
      for (int c = lane; c < columns; c += kAhead * 32) {
        T y[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          y[i] = T{};
          if (row >= 0 && c + i * 32 < columns) y[i] = in[c + i * 32];
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
          if (c + i * 32 < columns) out[c + i * 32] = y[i];
      }
    });
  }
}

__global__ void __launch_bounds__(kRowThreads) fork_kernel(const __grid_constant__ PoolProblem p) {
  extern __shared__ __align__(128) unsigned char memory[];
  __shared__ RingMemory rings;
  Ring ring(rings, memory, p.stage_bytes, p.status, kSiteCopy);
  unsigned char* const zeros = memory + kStages * kCopyWarps * p.stage_bytes;
  int *const slot = reinterpret_cast<int*>(zeros + p.stage_bytes), *const src = slot + p.n;
  const int tid = threadIdx.x;
  for (int i = tid; i < p.stage_bytes / 16; i += kRowThreads) reinterpret_cast<uint4*>(zeros)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async();
  griddep_wait();
  // marks and sources of pools that are not large come to shared memory at once: several passes go over them
  __shared__ uint8_t marks[kGroupSlots];
  __shared__ int sources[kGroupEntries];
  const bool small = p.slots <= kGroupSlots && p.n <= kGroupEntries;
  if (small) {
    for (int s = tid; s < p.slots; s += kRowThreads) marks[s] = p.live[s];
    for (int e = tid; e < p.n; e += kRowThreads) {
      const long long s = index_at(p.source, p.source64, e);
      sources[e] = s >= -1 && s < p.slots ? static_cast<int>(s) : -2;
    }
    __syncthreads();
  }
  const uint8_t* const live = small ? marks : p.live;
  auto source = [&](int e) { return small ? sources[e] : index_at(p.source, p.source64, e); };
  // the lowest n free slots
  const int each = (p.slots + kRowThreads - 1) / kRowThreads, s0 = min(p.slots, tid * each), s1 = min(p.slots, s0 + each);
  int free = 0;
  for (int s = s0; s < s1; ++s) free += !live[s];
  unsigned frees, total;
  const int before = block_scan(free, &frees);
  int at = before;
  for (int s = s0; s < s1 && at < p.n; ++s)
    if (!live[s]) slot[at++] = s;
  __syncthreads();
  // the entries that take one
  const int per = (p.n + kRowThreads - 1) / kRowThreads, e0 = min(p.n, tid * per), e1 = min(p.n, e0 + per);
  auto takes = [&](int e) {
    const long long s = source(e);
    return s == -1 || (s >= 0 && s < p.slots && live[s]);
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
        src[at] = static_cast<int>(source(e));
      }
      ++at;
    }
    if (blockIdx.x == 0) p.target[e] = got;
  }
  if (blockIdx.x == 0) {
    at = before;
    for (int s = s0; s < s1; ++s) p.after[s] = live[s] || at++ < moves;
  }
  __syncthreads();
  auto from = [&](int m) { return static_cast<long long>(src[m]); };
  auto to = [&](int m) { return slot[m]; };
  if (!p.together) {
    copy_rows(p, ring, zeros, moves, from, [](int) { return 1; }, [&](int c, int) { return slot[c]; }, moves, from, to);
    return;
  }
  // Together by their source, so that it is read once for up to kMostTargets of them: places by counting, in every CTA the same.
  int2* const chunk = reinterpret_cast<int2*>((reinterpret_cast<uintptr_t>(src + p.n) + 7) / 8 * 8);      // source; first place and how many
  int* const count = reinterpret_cast<int*>(chunk + p.n);                                                 // [slots + 1], by source + 1
  uint16_t *const order = reinterpret_cast<uint16_t*>(count + p.slots + 1), *const rank = order + p.n;
  for (int s = tid; s <= p.slots; s += kRowThreads) count[s] = 0;
  __syncthreads();
  for (int m = tid; m < moves; m += kRowThreads) {
    const int of = src[m];
    int earlier = 0;
#pragma unroll 8
    for (int j = 0; j < m; ++j) earlier += src[j] == of;
    rank[m] = static_cast<uint16_t>(earlier);
    atomicAdd(count + of + 1, 1);
  }
  __syncthreads();
  const int keys = p.slots + 1, share = (keys + kRowThreads - 1) / kRowThreads, k0 = min(keys, tid * share), k1 = min(keys, k0 + share);
  unsigned sums = 0;      // places and chunks of the sources in front
  for (int k = k0; k < k1; ++k) sums += count[k] | ((count[k] + kMostTargets - 1) / kMostTargets) << 16;
  sums = block_scan(sums, &total);
  const int chunks = total >> 16;
  for (int k = k0; k < k1; ++k) {
    const int c = count[k];
    for (int i = 0; i < c; i += kMostTargets) chunk[(sums >> 16) + i / kMostTargets] = make_int2(k - 1, ((sums & 0xffff) + i) << 8 | min(kMostTargets, c - i));
    count[k] = sums & 0xffff;
    sums += c | ((c + kMostTargets - 1) / kMostTargets) << 16;
  }
  __syncthreads();
  for (int m = tid; m < moves; m += kRowThreads) order[count[src[m] + 1] + rank[m]] = static_cast<uint16_t>(slot[m]);
  __syncthreads();
  copy_rows(p, ring, zeros, chunks, [&](int c) { return static_cast<long long>(chunk[c].x); }, [&](int c) { return chunk[c].y & 0xff; },
            [&](int c, int i) { return order[(chunk[c].y >> 8) + i]; }, moves, from, to);
}

__global__ void __launch_bounds__(kRowThreads) compact_kernel(const __grid_constant__ PoolProblem p) {
  extern __shared__ __align__(128) unsigned char memory[];
  __shared__ RingMemory rings;
  Ring ring(rings, memory, p.stage_bytes, p.status, kSiteCopy);
  uint16_t *const src = reinterpret_cast<uint16_t*>(memory + kStages * kCopyWarps * p.stage_bytes), *const dst = src + p.slots / 2;
  const int tid = threadIdx.x;
  griddep_wait();
  __shared__ uint8_t marks[kGroupSlots];
  const bool small = p.slots <= kGroupSlots;
  if (small) {
    for (int s = tid; s < p.slots; s += kRowThreads) marks[s] = p.live[s];
    __syncthreads();
  }
  const uint8_t* const live_at = small ? marks : p.live;
  const int each = (p.slots + kRowThreads - 1) / kRowThreads, s0 = min(p.slots, tid * each), s1 = min(p.slots, s0 + each);
  unsigned live = 0, total;
  for (int s = s0; s < s1; ++s) live += live_at[s] != 0;
  block_scan(live, &total);
  const int count = total;
  // those behind the place of the last live slot to be, and the holes in front of it: as many of one as of the other
  unsigned both = 0;
  for (int s = s0; s < s1; ++s) both += live_at[s] ? s >= count : (s < count ? 1u << 16 : 0u);
  const unsigned before = block_scan(both, &total);
  const int moves = total & 0xffff;
  int leave = before & 0xffff, hole = before >> 16;
  for (int s = s0; s < s1; ++s) {
    if (live_at[s]) {
      if (s >= count) src[leave++] = static_cast<uint16_t>(s);
    } else if (s < count) {
      dst[hole++] = static_cast<uint16_t>(s);
    }
  }
  __syncthreads();
  leave = before & 0xffff;
  for (int s = s0; s < s1; ++s) {
    long long to = -1;
    if (live_at[s]) to = s < count ? s : dst[leave++];
    if (static_cast<unsigned>(s) % gridDim.x == blockIdx.x) p.place[s] = to;
  }
  if (blockIdx.x == 0 && tid == 0) *p.live_count = count;
  auto from = [&](int m) { return static_cast<long long>(src[m]); };
  auto to = [&](int m) { return dst[m]; };
  copy_rows(p, ring, nullptr, moves, from, [](int) { return 1; }, [&](int c, int) { return dst[c]; }, moves, from, to);
}

// ------------------------------------------------------------------------------------------------------------------
// The tensors of a call that go into one launch, with rows of 16-byte multiples or of others; `groups`: how often each is counted.
static void take_states(const LetheGdnStates* s, int count, bool bulk, int strip, long long groups, StateTensors* out, long long* items) {
  long long n = 0;
  out->count = 0;
  for (int i = 0; i < count; ++i) {
    StateTensor t;
    t.data = static_cast<char*>(s[i].data);
    t.row = s[i].row_bytes;
    t.stride = s[i].stride;
    t.group = s[i].group_stride;
    const unsigned long long bits = reinterpret_cast<uintptr_t>(t.data) | t.row | t.stride | t.group;
    t.unit = 16;
    while (bits % t.unit) t.unit /= 2;
    if ((t.unit == 16) != bulk) continue;
    t.strip = strip;
    t.first = n;
    n += groups * ((t.row + strip - 1) / strip);
    out->t[out->count++] = t;
  }
  *items = n;
}
static int check_states(const LetheGdnStates* s, int count) {
  if (count < 0 || (count && !s)) return kErrNull;
  for (int i = 0; i < count; ++i) {
    if (!s[i].data) return kErrNull;
    if (s[i].row_bytes <= 0 || s[i].row_bytes > (1ll << 40)) return kErrDims;
  }
  return kOk;
}
template <typename Launch> static int in_launches(const LetheGdnStates* states, int count, Launch launch) {
  for (int i = 0; i == 0 || i < count; i += kMostTensors) {
    const int rc = launch(states + i, count - i < kMostTensors ? count - i : kMostTensors);
    if (rc != kOk) return rc;
  }
  return kOk;
}
constexpr int kPlainStrip = 2048;
// bytes of a strip, `most` or halves of it, so that there are `items` of `rows` rows of every tensor
static int balanced(const LetheGdnStates* s, int count, long long rows, int most, long long items) {
  long long bytes = 0;
  for (int i = 0; i < count; ++i) bytes += rows * s[i].row_bytes;
  int strip = most;
  while (strip >= 4096 && strip % 1024 == 0 && bytes / strip < items) strip /= 2;
  return strip;
}
static unsigned ctas_for(long long bulk, long long plain, int sms) {
  const long long p = (plain + kPlainWarps - 1) / kPlainWarps, n = bulk > p ? bulk : p;
  return static_cast<unsigned>(n < 1 ? 1 : n < sms ? n : sms);
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
  for (int i = 0; i < count; ++i)      // strips of a row are counted in 32 bits, those of all tensors in 64
    if (states[i].row_bytes > (1ll << 38) || states[i].row_bytes / 128 + 1 > (1ll << 57) / B) return kErrDims;
  DeviceGuard guard(states[0].data);
  if (!guard.ok) return kErrDevice;
  const int sms = sm_count();
  if (sms <= 0) return kErrDevice;
  static SmemAttr attr;
  if (attr.set(reorder_kernel, kAllBytes)) return kErrLaunch;
  const bool wide = W > 32;
  return in_launches(states, count, [&](const LetheGdnStates* s, int n) {
    ReorderProblem p = {};
    p.parents = parents;
    p.parents64 = parents_64;
    p.W = W;
    p.status = status;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (wide) {
      int part = 128;
      while (2 * part * W <= kGroupBytes) part *= 2;
      long long more;
      take_states(s, n, false, part, B, &p.plain, &p.plain_items);
      StateTensors& all = p.plain;      // those of 16-byte multiples behind them
      take_states(s, n, true, part, B, &p.bulk, &more);
      for (int i = 0; i < p.bulk.count; ++i) {
        all.t[all.count] = p.bulk.t[i];
        all.t[all.count++].first += p.plain_items;
      }
      p.plain_items += more;
      return launch_dependent(reorder_wide_kernel, dim3(static_cast<unsigned>(p.plain_items < kMostWideCtas ? p.plain_items : kMostWideCtas)), dim3(kRowThreads), kGroupBytes, st, p) == cudaSuccess ? kOk : kErrLaunch;
    }
    take_states(s, n, false, kPlainStrip, B, &p.plain, &p.plain_items);
    const int plain_bytes = p.plain_items ? kPlainWarps * W * 32 * 8 : 0;      // (units of 8 bytes at most)
    // fewer and larger rings for wide groups, whose strips share a stage; strips short enough for all rings
    p.copy_warps = W <= 8 ? kCopyWarps : W <= 16 ? kCopyWarps / 2 : 1;
    const int strip = balanced(s, n, B, 4 * kMostStage, 2LL * p.copy_warps * sms);
    take_states(s, n, true, strip, B, &p.bulk, &p.bulk_items);
    p.stage_bytes = p.bulk_items ? (kAllBytes - plain_bytes) / (kStages * p.copy_warps) / 512 * 512 : 0;
    if (p.stage_bytes * p.copy_warps > kMostStage * kCopyWarps) p.stage_bytes = kMostStage * kCopyWarps / p.copy_warps;
    return launch_dependent(reorder_kernel, dim3(ctas_for(p.bulk_items, p.plain_items, sms)), dim3(kRowThreads), kStages * p.copy_warps * p.stage_bytes + plain_bytes, st, p) == cudaSuccess ? kOk : kErrLaunch;
  });
}

static int pool_call(const LetheGdnStates* states, int count, long long slots, const uint8_t* live, lg::PoolProblem* p, bool fork, int lists,
                     long long most, int* status, void* stream) {
  using namespace lg;
  DeviceGuard guard(live);
  if (!guard.ok) return kErrDevice;
  const int sms = sm_count();
  if (sms <= 0) return kErrDevice;
  static SmemAttr attrs[2];
  if (attrs[fork].set(fork ? fork_kernel : compact_kernel, kAllBytes)) return kErrLaunch;
  p->live = live;
  p->slots = static_cast<int>(slots);
  p->status = status;
  const int stages = kStages * kCopyWarps + (fork ? 1 : 0), room = (kAllBytes - lists) / stages / 512 * 512;
  return in_launches(states, count, [&](const LetheGdnStates* s, int n) {
    p->stage_bytes = balanced(s, n, most, room < kMostStage ? room : kMostStage, 2LL * kCopyWarps * sms);
    take_states(s, n, true, p->stage_bytes, 1, &p->bulk, &p->bulk_strips);
    take_states(s, n, false, kPlainStrip, 1, &p->plain, &p->plain_strips);
    const unsigned grid = ctas_for(p->bulk_strips * most, p->plain_strips * most, sms);
    return launch_dependent(fork ? fork_kernel : compact_kernel, dim3(grid), dim3(kRowThreads), stages * p->stage_bytes + lists, static_cast<cudaStream_t>(stream), *p) == cudaSuccess ? kOk : kErrLaunch;
  });
}

extern "C" int lethe_gdn_fork_states(const LetheGdnStates* states, int32_t count, int64_t slots, const uint8_t* live, const void* source,
                                     int32_t source_64, int64_t n, int64_t* target, uint8_t* live_after, int32_t* status, void* stream) {
  using namespace lg;
  if (!live || !source || !target || !live_after || !status) return kErrNull;
  const int bad = check_states(states, count);
  if (bad) return bad;
  if (slots <= 0 || slots > kMostSlots || n <= 0 || n > kMostEntries) return kErrDims;
  if (reinterpret_cast<uintptr_t>(source) % (source_64 ? 8 : 4) || reinterpret_cast<uintptr_t>(target) % 8) return kErrAlign;
  // (one CTA writes the results while others still work out the plan)
  const long long source_bytes = n * (source_64 ? 8 : 4);
  if (meet(live_after, slots, live, slots) || meet(live_after, slots, source, source_bytes) || meet(target, 8 * n, live, slots) ||
      meet(target, 8 * n, source, source_bytes) || meet(target, 8 * n, live_after, slots))
    return kErrShared;
  PoolProblem p = {};
  p.source = source;
  p.source64 = source_64;
  p.n = static_cast<int>(n);
  p.target = reinterpret_cast<long long*>(target);
  p.after = live_after;
  // What L2 holds may be read once for each target.
  double bytes = 0;
  for (int i = 0; i < count; ++i) bytes += static_cast<double>(n) * states[i].row_bytes;
  p.together = bytes > kTogetherBytes && slots <= kGroupSlots && n <= kGroupEntries;
  return pool_call(states, count, slots, live, &p, true, fork_list_bytes(static_cast<int>(slots), p.n, p.together), n < slots ? n : slots, status, stream);
}

extern "C" int lethe_gdn_compact_states(const LetheGdnStates* states, int32_t count, int64_t slots, const uint8_t* live, int64_t* place,
                                        int64_t* live_count, int32_t* status, void* stream) {
  using namespace lg;
  if (!live || !place || !live_count || !status) return kErrNull;
  const int bad = check_states(states, count);
  if (bad) return bad;
  if (slots <= 0 || slots > kMostSlots) return kErrDims;
  if ((reinterpret_cast<uintptr_t>(place) | reinterpret_cast<uintptr_t>(live_count)) % 8) return kErrAlign;
  if (meet(place, 8 * slots, live, slots) || meet(live_count, 8, live, slots) || meet(live_count, 8, place, 8 * slots)) return kErrShared;
  PoolProblem p = {};
  p.place = reinterpret_cast<long long*>(place);
  p.live_count = reinterpret_cast<long long*>(live_count);
  return pool_call(states, count, slots, live, &p, false, 2 * static_cast<int>(slots), slots / 2, status, stream);
}
