// The element-wise gated recurrence h_t = e^{g_t} h_{t-1} + x_t (or + (1 - e^{g_t}) x_t), its backward, and one token of it.
//
// Bound by HBM: some 10 to 20 operations for every 8 bytes forward (bf16 x and h, fp32 g) and 14 backward.
//
// A CTA does a tile of kTokens tokens of kChannels channels of one sequence, read once and held in registers: a thread has kSteps
// tokens of four channels, its 16-lane group covers the channels, kGroups groups the tokens.  Every thread runs its own tokens from
// a zero state, the groups' results (sum of g, state) meet in shared memory and are folded in order, the tile gets the state in
// front of it from the tiles before (below), and every thread runs its tokens again from the state that it really starts from.
// The order of all sums is fixed, so two runs give the same bits.
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
  // e^g - 1 = g (1 + g/2 + g^2/6 + ... + g^6/5040): the first term left out is under 2e-9 of the result for |g| <= 1/4
  float s = fmaf(g, 1.f / 5040.f, 1.f / 720.f);
  s = fmaf(g, s, 1.f / 120.f);
  s = fmaf(g, s, 1.f / 24.f);
  s = fmaf(g, s, 1.f / 6.f);
  s = fmaf(g, s, 0.5f);
  s = fmaf(g, s, 1.f);
  const float m = -fabsf(g) * s;      // (-0 for both zeros)
  float e;      // 2 ulp and the rounding of the product: beyond -1/4 a memory is shorter than five tokens
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * 1.4426950408889634f));
  return g > -0.25f && g <= 0.f ? m : e;
}
__device__ __forceinline__ bool is_diff(float c) { return static_cast<int>(__float_as_uint(c)) < 0; }
// e^g h + x
__device__ __forceinline__ float decay_step(float c, float h, float x) {
  const float t = fmaf(c, h, x);
  return is_diff(c) ? h + t : t;
}
// coefficient of two steps, one after the other
__device__ __forceinline__ float decay_both(float c, float d) {
  if (is_diff(c) && is_diff(d)) {
    const float m = -fabsf(fmaf(c, d, c + d));
    return m >= -0.5f ? m : 1.f + m;
  }
  return (is_diff(c) ? 1.f + c : c) * (is_diff(d) ? 1.f + d : d);
}
__device__ __forceinline__ float forgotten(float c) { return is_diff(c) ? -c : 1.f - c; }      // 1 - e^g

struct LookBuffer {
  uint32_t* head;                   // ticket, and the word that lets everybody pass
  unsigned long long* word[3];      // of tiles, groups of tiles, groups of groups
};
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
  uint32_t seqs;          // B strips
  int* status;
  LookBuffer look;
};

// What a thread keeps from its first run over its tokens to its second: the compiler would keep everything that it formed there as
// well (fp32 copies, 1 - e^g), for twice the registers.
template <int TY>
__device__ __forceinline__ void forget_copies(Raw<TY, kPer> (&r)[kSteps]) {
#pragma unroll
  for (int s = 0; s < kSteps; ++s)
#pragma unroll
    for (int i = 0; i < Raw<TY, kPer>::kWords; ++i) asm volatile("" : "+r"(r[s].w[i]));
}
__device__ __forceinline__ void forget_copies(float (&c)[kSteps][kPer]) {
#pragma unroll
  for (int s = 0; s < kSteps; ++s)
#pragma unroll
    for (int j = 0; j < kPer; ++j) asm volatile("" : "+f"(c[s][j]));
}

// Four channels of one token, W neighbours at a time: as many as D, strides and alignment let be loaded at once.
template <int W>
__device__ __forceinline__ int channel_of(int lane, int j) { return (j / W * kLanes + lane) * W + j % W; }

// What a thread loads next lies in shared memory in places of its own, so that it is under way while the thread works on what it has
// in registers; nobody else reads it, so nothing but the thread's own wait stands between.  [step][piece][thread]: no bank conflicts.
template <int TY, int W> struct Staged {
  static constexpr int kBytes = W * elem_bytes(TY), kPieces = kPer / W, kWords = kBytes / 4;
  static constexpr bool kAsync = kBytes >= 4;      // (2 bytes are no asynchronous copy: loaded when they are wanted)
  alignas(16) uint32_t w[kAsync ? kSteps : 1][kPieces][kAsync ? kScanThreads : 1][kAsync ? kWords : 1];      // (a copy's two ends lie on a boundary of its size)

  // `base`: the tensor, an address that is good where nothing is read
  __device__ __forceinline__ void fetch(const typename Elem<TY>::T* p, const void* base, long long stride, int lane, int live, int room) {
    if constexpr (kAsync) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
          const int ch = channel_of<W>(lane, i * W);
          const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(&w[s][i][threadIdx.x][0]));
          const bool there = s < live && ch < room;      // zeros otherwise
          const void* from = there ? p + s * stride + ch : base;
          if constexpr (kBytes == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
          else
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(kBytes), "r"(there ? kBytes : 0) : "memory");
        }
    }
  }
  __device__ __forceinline__ void take(Raw<TY, kPer> (&r)[kSteps], const typename Elem<TY>::T* p, long long stride, int lane, int live, int room) const {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      if constexpr (kAsync) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
          for (int k = 0; k < kWords; ++k) r[s].w[i * kWords + k] = w[s][i][threadIdx.x][k];
      } else {
        r[s].zero();
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (s < live && channel_of<W>(lane, j) < room) raw_put(r[s], j, __ldg(p + s * stride + channel_of<W>(lane, j)));
      }
    }
  }
};
template <int TY, int W>
__device__ __forceinline__ void store_token(const Raw<TY, kPer>& r, typename Elem<TY>::T* p, int lane, int room) {
  constexpr int kBytes = W * elem_bytes(TY), kWords = kBytes / 4;
#pragma unroll
  for (int i = 0; i < kPer / W; ++i) {
    const int ch = channel_of<W>(lane, i * W);
    if (ch >= room) continue;
    uint32_t* d = reinterpret_cast<uint32_t*>(p + ch);
    if constexpr (kWords == 4) *reinterpret_cast<uint4*>(d) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    else if constexpr (kWords == 2) *reinterpret_cast<uint2*>(d) = make_uint2(r.w[i * 2], r.w[i * 2 + 1]);
    else if constexpr (kWords == 1) *d = r.w[i];
    else p[ch] = raw_take(r, i);
  }
}
template <int TY>
__device__ __forceinline__ Raw<TY, kPer> packed(const float (&v)[kPer]) {
  Raw<TY, kPer> r;
  r.set2(0, v[0], v[1]);
  r.set2(2, v[2], v[3]);
  return r;
}

// ---------------------------------------------------------------------------------------------
// What a tile hands on.  The state in front of a tile depends on all tiles before it; a tile leaves its own part, (coefficient
// of its decay, state from zero), in the work buffer as soon as it has it, 64 bits per channel, stored and loaded as one, so a word
// that is there is whole and needs no flag or fence beside it.  Unwritten words are all ones (the buffer is set so in front of the kernel).
//
// Three levels keep what a tile has to read at 31 words: the tiles of its group of 16 in front of it, the groups of its 16 groups in
// front of it (the last tile of a group leaves that word, from the group's words alone), and the state behind the 256 tiles before
// those (left by the last of them).  The order of the fold is that of the tokens whoever comes first.
//
// Tiles are taken by ticket, so a tile waits only for tiles whose CTAs run already and wait for earlier ones only.  Waits are
// bounded all the same: one that runs out leaves a code in the status word and lets everybody pass.
// ---------------------------------------------------------------------------------------------
constexpr int kFan = 16;
constexpr long long kLookLimitCycles = 2000000000LL;      // about one second
enum : int { kSiteLook = 900 };

constexpr size_t kLookHead = 128;
struct LookSizes {
  size_t count[3];
  size_t bytes() const { return kLookHead + (count[0] + count[1] + count[2]) * kChannels * 8; }
};
static LookSizes look_sizes(long long seqs, long long tiles) {
  if (tiles <= 1) return {{0, 0, 0}};
  const long long groups = (tiles + kFan - 1) / kFan, supers = (groups + kFan - 1) / kFan;
  return {{static_cast<size_t>(seqs * tiles), static_cast<size_t>(seqs * groups), static_cast<size_t>(seqs * supers)}};
}

__device__ __forceinline__ unsigned long long look_load(const unsigned long long* p) {
  unsigned long long v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void look_store(unsigned long long* p, float coef, float state) {
  unsigned long long v = (static_cast<unsigned long long>(__float_as_uint(state)) << 32) | __float_as_uint(coef);
  if (v == ~0ull) v = 0x7fffffff7fffffffull;      // (another NaN)
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}
__device__ __noinline__ unsigned long long look_wait(const unsigned long long* p, uint32_t* head, int* status) {
  const long long t0 = clock64();
  for (int n = 1;; ++n) {
    const unsigned long long v = look_load(p);
    if (v != ~0ull) return v;
    if (n % 32) continue;
    if (*reinterpret_cast<volatile uint32_t*>(head + 1) == 0u) return 0;
    if (clock64() - t0 > kLookLimitCycles) {
      atomicCAS(status, 0, kSiteLook);
      *reinterpret_cast<volatile uint32_t*>(head + 1) = 0u;
      return 0;
    }
  }
}

struct LookShared {
  float2 part[2 * kFan - 1][kChannels];      // (coefficient, state): groups, then tiles, in front
  float base[kChannels];                     // state behind the 256 tiles before
};
struct ScanShared {
  float2 part[kGroups][kChannels];      // per group of tokens: (coefficient of its whole decay, state from zero)
  float sum[kGroups][kChannels];        // sum of its g
  float start[kGroups][kChannels];      // state in front of it
  LookShared look;
  uint32_t ticket[2];
};
struct ScanSharedBackward : ScanShared {
  float back[kGroups][kChannels];       // per group the gradient that leaves it towards earlier tokens, from zero
  float end[kGroups][kChannels];        // the gradient that comes into it
};
template <int XT, int GT, int W> struct ForwardShared : ScanShared {
  Staged<XT, W> x;
  Staged<GT, W> g;
};
static_assert(alignof(Staged<LETHE_F32, 4>) == 16 && sizeof(Staged<LETHE_BF16, 4>) % 16 == 0, "asynchronous copies of 16 bytes");
template <int XT, int GT, int W> struct BackwardShared : ScanSharedBackward {
  Staged<XT, W> x, d;
  Staged<GT, W> g;
};

// Where tile number `i` (in the order of the fold) of sequence `seq` stands among the three levels.
struct LookPlace {
  LookBuffer buf;
  long long group0, tile0;      // first words of its level: groups of its super, tiles of its group
  long long super;              // its super's word
  int n_groups, n_tiles;        // how many in front of it
  bool first_super, last;       // no tiles in front of its super; no tile behind it
  __device__ LookPlace(const LookBuffer& b, long long seq, int tiles, int i) : buf(b) {
    const int groups = (tiles + kFan - 1) / kFan, supers = (groups + kFan - 1) / kFan;
    const int sup = i / (kFan * kFan);
    n_groups = i / kFan % kFan;
    n_tiles = i % kFan;
    group0 = seq * groups + sup * kFan;
    tile0 = seq * tiles + (i - n_tiles);
    super = seq * supers + sup;
    first_super = sup == 0;
    last = i == tiles - 1;
  }
  __device__ unsigned long long* at(int level, long long n, int ch) const { return buf.word[level] + n * kChannels + ch; }
};

// All threads.  Leaves what the fold reads in `l`; in between the last tile of a group leaves the group's word: `coef`, `state` of
// threads below kChannels are the tile's own.
__device__ __forceinline__ void look_fetch(LookShared& l, const LookPlace& p, float coef, float state, int* status) {
  const int ch = threadIdx.x % kChannels, q = threadIdx.x / kChannels;
  constexpr int kQ = kScanThreads / kChannels, kEach = (kFan + kQ - 1) / kQ;
  const auto as_pair = [](unsigned long long v) { return make_float2(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32))); };
  unsigned long long t[kEach], g[kEach], b = 0;
#pragma unroll
  for (int m = 0; m < kEach; ++m) {
    const int k = q + m * kQ;
    if (k < p.n_tiles) t[m] = look_load(p.at(0, p.tile0 + k, ch));
  }
#pragma unroll
  for (int m = 0; m < kEach; ++m) {
    const int k = q + m * kQ;
    if (k < p.n_groups) g[m] = look_load(p.at(1, p.group0 + k, ch));
  }
  if (q == 0 && !p.first_super) b = look_load(p.at(2, p.super - 1, ch));
#pragma unroll
  for (int m = 0; m < kEach; ++m) {
    const int k = q + m * kQ;
    if (k < p.n_tiles) {
      if (t[m] == ~0ull) t[m] = look_wait(p.at(0, p.tile0 + k, ch), p.buf.head, status);
      l.part[p.n_groups + k][ch] = as_pair(t[m]);
    }
  }
  if (p.n_tiles == kFan - 1 && !p.last) {      // (the same for all threads of a CTA)
    __syncthreads();
    if (q == 0) {
      float gc = -0.f, gh = 0.f;
      for (int k = 0; k < kFan - 1; ++k) {
        const float2 a = l.part[p.n_groups + k][ch];
        gc = decay_both(gc, a.x);
        gh = decay_step(a.x, gh, a.y);
      }
      look_store(p.at(1, p.group0 + p.n_groups, ch), decay_both(gc, coef), decay_step(coef, gh, state));
    }
  }
#pragma unroll
  for (int m = 0; m < kEach; ++m) {
    const int k = q + m * kQ;
    if (k < p.n_groups) {
      if (g[m] == ~0ull) g[m] = look_wait(p.at(1, p.group0 + k, ch), p.buf.head, status);
      l.part[k][ch] = as_pair(g[m]);
    }
  }
  if (q == 0 && !p.first_super) {
    if (b == ~0ull) b = look_wait(p.at(2, p.super - 1, ch), p.buf.head, status);
    l.base[ch] = as_pair(b).y;
  }
  __syncthreads();
}
// Threads below kChannels: the state in front of the tile; `first`: that in front of the first tile.
__device__ __forceinline__ float look_fold(const LookShared& l, const LookPlace& p, float first) {
  float carry = p.first_super ? first : l.base[threadIdx.x];
  for (int k = 0; k < p.n_groups + p.n_tiles; ++k) {
    const float2 a = l.part[k][threadIdx.x];
    carry = decay_step(a.x, carry, a.y);
  }
  return carry;
}

// Where a tile lies.
struct TilePlace {
  long long seq, b, ch0, t0;      // sequence (a strip of one), batch, first channel, first token of this thread
  int tile, room, live;           // channels of the strip; tokens of this thread (0 and less: none)
  __device__ __forceinline__ TilePlace(const DiagProblem& p, uint32_t ticket, int grp, bool backwards) {
    const uint32_t order = ticket / p.seqs;
    seq = ticket - order * p.seqs;
    tile = backwards ? p.tiles - 1 - static_cast<int>(order) : static_cast<int>(order);
    const uint32_t s = static_cast<uint32_t>(seq);
    b = s / static_cast<uint32_t>(p.strips);
    ch0 = static_cast<long long>(s % static_cast<uint32_t>(p.strips)) * kChannels;
    room = static_cast<int>(p.D - ch0 < kChannels ? p.D - ch0 : kChannels);
    t0 = static_cast<long long>(tile) * kTokens + grp * kSteps;
    live = static_cast<int>(p.L - t0 < kSteps ? p.L - t0 : kSteps);
  }
};

// The CTAs take tiles until there are none; a CTA's tickets ascend, and it takes the next one while it works on a tile: the tile of the
// lowest ticket that is not done is the one that its CTA works on, so somebody always can go on.
template <int XT, int GT, int W, bool COMP>
__global__ void __launch_bounds__(kScanThreads, 2) diag_forward_kernel(const DiagProblem p) {
  using X = typename Elem<XT>::T;
  using G = typename Elem<GT>::T;
  extern __shared__ __align__(16) unsigned char smem[];
  auto& sh = *reinterpret_cast<ForwardShared<XT, GT, W>*>(smem);
  const int lane = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const uint32_t total = p.seqs * static_cast<uint32_t>(p.tiles);
  const auto take_ticket = [&](uint32_t have) { return p.tiles > 1 ? atomicAdd(p.look.head, 1u) + 1u : have + gridDim.x; };
  const auto x_at = [&](const TilePlace& t) { return static_cast<const X*>(p.x) + t.b * p.x_batch + t.t0 * p.x_token + t.ch0; };
  const auto g_at = [&](const TilePlace& t) { return static_cast<const G*>(p.g) + t.b * p.g_batch + t.t0 * p.g_token + t.ch0; };
  const auto fetch = [&](uint32_t ticket) {
    if (ticket < total) {
      const TilePlace t(p, ticket, grp, false);
      sh.x.fetch(x_at(t), p.x, p.x_token, lane, t.live, t.room);
      sh.g.fetch(g_at(t), p.g, p.g_token, lane, t.live, t.room);
    }
  };
  if (threadIdx.x == 0) {
    const uint32_t first = p.tiles > 1 ? take_ticket(0) : blockIdx.x;
    sh.ticket[0] = first;
    sh.ticket[1] = take_ticket(first);
  }
  __syncthreads();
  uint32_t ticket = sh.ticket[0];
  fetch(ticket);
  for (int turn = 0; ticket < total; turn ^= 1) {
    const TilePlace at(p, ticket, grp, false);
    const int room = at.room, live = at.live;
    Raw<XT, kPer> xr[kSteps];
    float c[kSteps][kPer], sum[kPer], st[kPer];
    const uint32_t next = sh.ticket[turn ^ 1];
    uint32_t after = 0;
    {
      Raw<GT, kPer> gr[kSteps];
      asm volatile("cp.async.wait_all;" ::: "memory");
      sh.x.take(xr, x_at(at), p.x_token, lane, live, room);
      sh.g.take(gr, g_at(at), p.g_token, lane, live, room);
      fetch(next);
      if (threadIdx.x == 0) after = take_ticket(next);
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
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int ch = channel_of<W>(lane, j);
      sh.part[grp][ch] = make_float2(decay_coef(sum[j]), st[j]);
      sh.sum[grp][ch] = sum[j];
    }
    forget_copies(xr);
    forget_copies(c);
    __syncthreads();
    if (threadIdx.x == 0) sh.ticket[turn] = after;      // (read behind the next barriers)
    const int ch = threadIdx.x;      // of threads below kChannels
    float carry = 0.f;
    if (ch < room && p.h0) carry = p.h0[at.b * p.D + at.ch0 + ch];
    if (p.tiles > 1) {
      const LookPlace look(p.look, at.seq, p.tiles, at.tile);
      float tc = -0.f, th = 0.f;
      if (ch < kChannels) {
        float ts = 0.f;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
          const float2 a = sh.part[i][ch];
          ts += sh.sum[i][ch];
          th = decay_step(a.x, th, a.y);
        }
        tc = decay_coef(ts);
        if (!look.last) look_store(look.at(0, look.tile0 + look.n_tiles, ch), tc, th);
      }
      look_fetch(sh.look, look, tc, th, p.status);
      if (ch < kChannels) {
        carry = look_fold(sh.look, look, carry);
        if (look.n_tiles == kFan - 1 && look.n_groups == kFan - 1 && !look.last) look_store(look.at(2, look.super, ch), 0.f, decay_step(tc, carry, th));
      }
    }
    if (ch < kChannels) {
      if (p.states && ch < room) p.states[(at.b * p.tiles + at.tile) * p.D + at.ch0 + ch] = carry;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        sh.start[i][ch] = carry;
        const float2 a = sh.part[i][ch];
        carry = decay_step(a.x, carry, a.y);
      }
      if (p.hT && ch < room && at.tile == p.tiles - 1) p.hT[at.b * p.D + at.ch0 + ch] = carry;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPer; ++j) st[j] = sh.start[grp][channel_of<W>(lane, j)];
    X* h = static_cast<X*>(p.h) + (at.b * p.L + at.t0) * p.D + at.ch0;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const float u = COMP ? xr[s].get(j) * forgotten(c[s][j]) : xr[s].get(j);
        st[j] = decay_step(c[s][j], st[j], u);
      }
      if (s < live) store_token<XT, W>(packed<XT>(st), h + s * p.D, lane, room);
    }
    ticket = next;
  }
}

template <int XT, int GT, int W, bool COMP>
__global__ void __launch_bounds__(kScanThreads, 2) diag_backward_kernel(const DiagProblem p) {
  using X = typename Elem<XT>::T;
  using G = typename Elem<GT>::T;
  extern __shared__ __align__(16) unsigned char smem[];
  auto& sh = *reinterpret_cast<BackwardShared<XT, GT, W>*>(smem);
  const int lane = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const uint32_t total = p.seqs * static_cast<uint32_t>(p.tiles);
  const auto take_ticket = [&](uint32_t have) { return p.tiles > 1 ? atomicAdd(p.look.head, 1u) + 1u : have + gridDim.x; };
  const auto x_at = [&](const TilePlace& t) { return static_cast<const X*>(p.x) + t.b * p.x_batch + t.t0 * p.x_token + t.ch0; };
  const auto g_at = [&](const TilePlace& t) { return static_cast<const G*>(p.g) + t.b * p.g_batch + t.t0 * p.g_token + t.ch0; };
  const auto d_at = [&](const TilePlace& t) { return static_cast<const X*>(p.d_h) + t.b * p.d_batch + t.t0 * p.d_token + t.ch0; };
  const auto fetch = [&](uint32_t ticket) {
    if (ticket < total) {
      const TilePlace t(p, ticket, grp, true);
      sh.x.fetch(x_at(t), p.x, p.x_token, lane, t.live, t.room);
      sh.g.fetch(g_at(t), p.g, p.g_token, lane, t.live, t.room);
      if (p.d_h) sh.d.fetch(d_at(t), p.d_h, p.d_token, lane, t.live, t.room);
    }
  };
  if (threadIdx.x == 0) {
    const uint32_t first = p.tiles > 1 ? take_ticket(0) : blockIdx.x;
    sh.ticket[0] = first;
    sh.ticket[1] = take_ticket(first);
  }
  __syncthreads();
  uint32_t ticket = sh.ticket[0];
  fetch(ticket);
  for (int turn = 0; ticket < total; turn ^= 1) {
    const TilePlace at(p, ticket, grp, true);
    const int room = at.room, live = at.live;
    Raw<XT, kPer> xr[kSteps], dr[kSteps];
    float c[kSteps][kPer], st[kPer], e[kPer];
    const uint32_t next = sh.ticket[turn ^ 1];
    uint32_t after = 0;
    {
      Raw<GT, kPer> gr[kSteps];
      float sum[kPer];
      asm volatile("cp.async.wait_all;" ::: "memory");
      sh.x.take(xr, x_at(at), p.x_token, lane, live, room);
      sh.g.take(gr, g_at(at), p.g_token, lane, live, room);
      if (p.d_h) {
        sh.d.take(dr, d_at(at), p.d_token, lane, live, room);
      } else {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) dr[s].zero();
      }
      fetch(next);
      if (threadIdx.x == 0) after = take_ticket(next);
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
        const int ch = channel_of<W>(lane, j);
        sh.part[grp][ch] = make_float2(decay_coef(sum[j]), st[j]);
        sh.sum[grp][ch] = sum[j];
        sh.back[grp][ch] = e[j];
      }
    }
    forget_copies(xr);
    forget_copies(dr);
    forget_copies(c);
    __syncthreads();
    if (threadIdx.x == 0) sh.ticket[turn] = after;
    const int ch = threadIdx.x, ch2 = threadIdx.x - kChannels;      // the gradient is folded by threads below kChannels, the state by the next ones
    float carry = 0.f;
    if (ch < room && p.dhT) carry = p.dhT[at.b * p.D + at.ch0 + ch];
    if (ch2 >= 0 && ch2 < kChannels) {
      float s0 = ch2 < room ? p.states[(at.b * p.tiles + at.tile) * p.D + at.ch0 + ch2] : 0.f;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        sh.start[i][ch2] = s0;
        const float2 a = sh.part[i][ch2];
        s0 = decay_step(a.x, s0, a.y);
      }
    }
    if (p.tiles > 1) {
      const LookPlace look(p.look, at.seq, p.tiles, p.tiles - 1 - at.tile);
      float tc = -0.f, te = 0.f;
      if (ch < kChannels) {
        float ts = 0.f;
#pragma unroll
        for (int i = kGroups - 1; i >= 0; --i) {
          ts += sh.sum[i][ch];
          te = decay_step(sh.part[i][ch].x, te, sh.back[i][ch]);
        }
        tc = decay_coef(ts);
        if (!look.last) look_store(look.at(0, look.tile0 + look.n_tiles, ch), tc, te);
      }
      look_fetch(sh.look, look, tc, te, p.status);
      if (ch < kChannels) {
        carry = look_fold(sh.look, look, carry);
        if (look.n_tiles == kFan - 1 && look.n_groups == kFan - 1 && !look.last) look_store(look.at(2, look.super, ch), 0.f, decay_step(tc, carry, te));
      }
    }
    if (ch < kChannels) {
#pragma unroll
      for (int i = kGroups - 1; i >= 0; --i) {
        sh.end[i][ch] = carry;
        carry = decay_step(sh.part[i][ch].x, carry, sh.back[i][ch]);
      }
      if (p.dh0 && ch < room && at.tile == 0) p.dh0[at.b * p.D + at.ch0 + ch] = carry;
    }
    __syncthreads();
    float before[kSteps][kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      st[j] = sh.start[grp][channel_of<W>(lane, j)];
      e[j] = sh.end[grp][channel_of<W>(lane, j)];
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const float xv = xr[s].get(j);
        before[s][j] = COMP ? st[j] - xv : st[j];
        st[j] = decay_step(c[s][j], st[j], COMP ? xv * forgotten(c[s][j]) : xv);
      }
    X* dx = static_cast<X*>(p.dx) + (at.b * p.L + at.t0) * p.D + at.ch0;
    G* dg = static_cast<G*>(p.dg) + (at.b * p.L + at.t0) * p.D + at.ch0;
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
      if (s < live) {
        if (p.dx) store_token<XT, W>(packed<XT>(vx), dx + s * p.D, lane, room);
        if (p.dg) store_token<GT, W>(packed<GT>(vg), dg + s * p.D, lane, room);
      }
    }
    ticket = next;
  }
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

// One token: state and h, four neighbouring channels a thread (W = 4) or one.
template <int XT, int GT, int W, bool COMP>
__global__ void __launch_bounds__(256) diag_step_kernel(const StepProblem p) {
  using X = typename Elem<XT>::T;
  using G = typename Elem<GT>::T;
  constexpr int N = W == kPer ? kPer : 1;
  const long long b = blockIdx.x / p.blocks, at = (static_cast<long long>(blockIdx.x % p.blocks) * 256 + threadIdx.x) * N;
  if (at >= p.D) return;
  const X* x = static_cast<const X*>(p.x) + b * p.x_batch + at;
  const G* g = static_cast<const G*>(p.g) + b * p.g_batch + at;
  X* h = static_cast<X*>(p.h) + b * p.D + at;
  float* st = p.state + b * p.D + at;
  if constexpr (N > 1) {
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

// f(XT, GT, W, COMP) as template arguments
template <typename F>
static int by_type(int xt, int gt, int w, bool comp, F&& f) {
  const auto flags = [&](auto x, auto g) {
    const auto last = [&](auto n) { return comp ? f(x, g, n, std::true_type()) : f(x, g, n, std::false_type()); };
    if (w == 4) return last(std::integral_constant<int, 4>());
    if (w == 2) return last(std::integral_constant<int, 2>());
    return last(std::integral_constant<int, 1>());
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
  if (strips > INT32_MAX || a->B > INT32_MAX / strips || tiles > INT32_MAX / (a->B * strips)) return kErrDims;
  *p = {a->B, a->L, a->D, a->x, a->x_batch, a->x_token, a->g, a->g_batch, a->g_token, a->h0, a->h, a->hT, a->states, a->d_h, a->d_h_batch,
        a->d_h_token, a->dhT, a->dx, a->dg, a->dh0, static_cast<int>(tiles), static_cast<int>(strips), static_cast<uint32_t>(a->B * strips), a->status, {}};
  if (tiles > 1) {
    if (!a->work) return kErrNull;
    if (reinterpret_cast<uintptr_t>(a->work) & 15) return kErrAlign;
    const LookSizes n = look_sizes(p->seqs, tiles);
    if (a->work_bytes < n.bytes()) return kErrWorkspace;
    p->look.head = static_cast<uint32_t*>(a->work);
    p->look.word[0] = reinterpret_cast<unsigned long long*>(static_cast<char*>(a->work) + kLookHead);
    for (int i = 1; i < 3; ++i) p->look.word[i] = p->look.word[i - 1] + n.count[i - 1] * kChannels;
  }
  return kOk;
}
// elements that can be moved at once
template <typename F>
static int widest(F&& fits) { return fits(4) ? 4 : fits(2) ? 2 : 1; }

template <typename Shared>
static int launch_scan_tiles(void (*kern)(DiagProblem), const DiagProblem& p, SmemAttr& attr, cudaStream_t st) {
  if (int e = attr.set(kern, sizeof(Shared))) return e;
  // all ones: no word is there yet, and the ticket before the first
  if (p.tiles > 1 && cudaMemsetAsync(p.look.head, 0xff, look_sizes(p.seqs, p.tiles).bytes(), st) != cudaSuccess) return kErrLaunch;
  const uint32_t total = p.seqs * static_cast<uint32_t>(p.tiles), room = 2u * static_cast<uint32_t>(sm_count());
  kern<<<total < room ? total : room, kScanThreads, sizeof(Shared), st>>>(p);
  return launched();
}

}  // namespace lg

extern "C" size_t lethe_gdn_diag_states_bytes(int64_t B, int64_t L, int64_t D) {
  using namespace lg;
  if (B <= 0 || L <= 0 || D <= 0) return 0;
  return static_cast<size_t>(B) * ((L + kTokens - 1) / kTokens) * D * sizeof(float);
}
extern "C" size_t lethe_gdn_diag_work_bytes(int64_t B, int64_t L, int64_t D) {
  using namespace lg;
  if (B <= 0 || L <= kTokens || D <= 0) return 0;
  return look_sizes(B * ((D + kChannels - 1) / kChannels), (L + kTokens - 1) / kTokens).bytes();
}

extern "C" int lethe_gdn_diag_forward(const LetheGdnDiagArgs* a, void* stream) {
  using namespace lg;
  DiagProblem p;
  if (int e = diag_problem(a, &p, false)) return e;
  DeviceGuard guard(a->x);
  if (!guard.ok) return kErrDevice;
  const int w = widest([&](int n) {
    return a->D % n == 0 && on_boundary(a->x, a->x_type, n, a->x_batch, a->x_token) && on_boundary(a->g, a->g_type, n, a->g_batch, a->g_token) &&
           on_boundary(a->h, a->x_type, n);
  });
  return by_type(a->x_type, a->g_type, w, a->complement != 0, [&](auto x, auto g, auto n, auto c) {
    static SmemAttr attr;
    return launch_scan_tiles<ForwardShared<x.value, g.value, n.value>>(diag_forward_kernel<x.value, g.value, n.value, c.value>, p, attr, static_cast<cudaStream_t>(stream));
  });
}

extern "C" int lethe_gdn_diag_backward(const LetheGdnDiagArgs* a, void* stream) {
  using namespace lg;
  DiagProblem p;
  if (int e = diag_problem(a, &p, true)) return e;
  DeviceGuard guard(a->x);
  if (!guard.ok) return kErrDevice;
  const int w = widest([&](int n) {
    return a->D % n == 0 && on_boundary(a->x, a->x_type, n, a->x_batch, a->x_token) && on_boundary(a->g, a->g_type, n, a->g_batch, a->g_token) &&
           on_boundary(a->d_h, a->x_type, n, a->d_h_batch, a->d_h_token) && on_boundary(a->dx, a->x_type, n) && on_boundary(a->dg, a->g_type, n);
  });
  return by_type(a->x_type, a->g_type, w, a->complement != 0, [&](auto x, auto g, auto n, auto c) {
    static SmemAttr attr;
    return launch_scan_tiles<BackwardShared<x.value, g.value, n.value>>(diag_backward_kernel<x.value, g.value, n.value, c.value>, p, attr, static_cast<cudaStream_t>(stream));
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
  return by_type(a->x_type, a->g_type, vec ? kPer : 1, a->complement != 0, [&](auto x, auto g, auto n, auto c) {
    diag_step_kernel<x.value, g.value, n.value == kPer ? kPer : 1, c.value>
        <<<static_cast<unsigned>(p.B * blocks), 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return launched();
  });
}
