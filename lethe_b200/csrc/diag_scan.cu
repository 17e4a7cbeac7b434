// The element-wise gated recurrence h_t = e^{g_t} h_{t-1} + x_t (or + (1 - e^{g_t}) x_t), its backward, and one token of it.
//
// Bound by HBM on paper: 8 bytes an element forward (bf16 x and h, fp32 g), 14 backward.  Measured (B1 L65536 D2048): 226 us forward, 0.73 of the
// measured copy bandwidth, 425 backward, 0.68; without any tile waiting for another (a tile a sequence: 1024 of 128 tokens forward, 2048 of 64
// backward) 210 and 403, so most of what is missing is the runs themselves, some 33 and 60 operations an element by 16 warps of an SM, not
// the handing on.  With the complement 246 and 505: its backward holds a value more for every step and spills 32 to 72 bytes a thread in 16 bits.
//
// A CTA does tiles, 16 groups of tokens x 64 channels of one sequence, each read once: a thread has 3 to 8 tokens of four channels, its
// 16-lane group covers the channels.  Every thread runs its own tokens from a zero state, the groups' results (sum of g, state) meet in
// shared memory and are folded in order, the tile gets the state in front of it from the tiles before (below), and every thread runs
// its tokens again from the state that it really starts from.  The order of all sums is fixed, so two runs give the same bits.
//
// The decay.  With memories of thousands of tokens e^g lies next to one, and fp32 rounds it by up to 2^-25: over n tokens the
// state is off by up to n times that, always to the same side where g is constant.  So below |g| = 1/4 the step is taken with
// c = e^g - 1 from its Taylor series, h + (c h + x): c is exact to a rounding of its own, and what is left is the rounding of
// the sum, which is even.  Beyond, where a memory is a few tokens, it is e^g h + x.  Both are one fused multiply-add with a
// coefficient whose sign bit says whether h is added (c <= -0) or not (e^g >= +0).  Decays of several tokens are kept as sums of g.
#include <type_traits>

#include "diag_look.cuh"
#include "elem.cuh"
#include "host_util.h"

namespace lg {

constexpr int kLanes = 16, kPer = 4, kChannels = kLanes * kPer;      // a strip of channels
constexpr int kPacked = 16;      // among the widths of the kernels: four channels at once, several batches in a strip
constexpr int kGroups = 16, kRunners = kLanes * kGroups;              // threads that hold a tile
constexpr int kPublisher = kRunners, kLooker = kPublisher + kChannels;  // first threads of those that hand on and of those that look back
constexpr int kScanThreads = kLooker + kChannels;
// Tokens of a thread: what two tiles of two CTAs take in shared memory decides.  The forward leaves a state for every tile of the backward.
constexpr int forward_steps(int xt) { return xt == LETHE_F32 ? 6 : 8; }
constexpr int backward_steps(int xt) { return forward_steps(xt) / 2; }

// whether the step over the log decay g is taken with the difference: -1/4 < g <= -0 (as whole numbers, negative floats are ordered
// backwards; +0 has the coefficient one)
__device__ __forceinline__ bool by_diff(float g) { return __float_as_int(g) < static_cast<int>(0xbe800000u); }
// coefficient of that step
__device__ __forceinline__ float decay_coef(float g) {
  // e^g - 1 = g (1 + g/2 + g^2/6 + ... + g^5/720): the first term left out is under 5e-8 of the result
  float s = fmaf(g, 1.f / 720.f, 1.f / 120.f);
  s = fmaf(g, s, 1.f / 24.f);
  s = fmaf(g, s, 1.f / 6.f);
  s = fmaf(g, s, 0.5f);
  s = fmaf(g, s, 1.f);
  float e;      // 2 ulp and the rounding of the product: beyond -1/4 a memory is shorter than five tokens
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * 1.4426950408889634f));
  return by_diff(g) ? g * s : e;
}
// the same for two at a time, in place: c[i] becomes the coefficient over c[i]
__device__ __forceinline__ void decay_coefs(float& g0, float& g1) {
  const F2 g = f2(g0, g1);
  F2 s = fma2(g, f2(1.f / 720.f), f2(1.f / 120.f));
  s = fma2(g, s, f2(1.f / 24.f));
  s = fma2(g, s, f2(1.f / 6.f));
  s = fma2(g, s, f2(0.5f));
  s = g * fma2(g, s, f2(1.f));
  const F2 t = g * f2(1.4426950408889634f);
  float e0, e1;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(lo(t)));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(hi(t)));
  g0 = by_diff(g0) ? lo(s) : e0;
  g1 = by_diff(g1) ? hi(s) : e1;
}
__device__ __forceinline__ bool is_diff(float c) { return static_cast<int>(__float_as_uint(c)) < 0; }
// e^g h + x
__device__ __forceinline__ float decay_step(float c, bool diff, float h, float x) {
  const float t = fmaf(c, h, x);
  return diff ? h + t : t;
}
__device__ __forceinline__ float decay_step(float c, float h, float x) { return decay_step(c, is_diff(c), h, x); }
__device__ __forceinline__ void add_to(float& a0, float& a1, float b0, float b1) {
  const F2 s = f2(a0, a1) + f2(b0, b1);
  a0 = lo(s);
  a1 = hi(s);
}
// two steps side by side
__device__ __forceinline__ void decay_steps(float c0, float c1, bool diff0, bool diff1, float& h0, float& h1, float x0, float x1) {
  const F2 t = fma2(f2(c0, c1), f2(h0, h1), f2(x0, x1));
  h0 = diff0 ? h0 + lo(t) : lo(t);
  h1 = diff1 ? h1 + hi(t) : hi(t);
}
// the same without x
__device__ __forceinline__ void decay_over(float c0, float c1, float& h0, float& h1) {
  const F2 t = f2(c0, c1) * f2(h0, h1);
  h0 = is_diff(c0) ? h0 + lo(t) : lo(t);
  h1 = is_diff(c1) ? h1 + hi(t) : hi(t);
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
  int tiles, strips;      // tiles of tokens, strips of kChannels channels
  long long records;      // states of a sequence that the forward keeps: one for every tile of the backward
  uint32_t seqs;          // strips of all batches: B strips, or fewer where a strip holds `pack` batches of D <= 32 channels
  int pack;
  size_t look_bytes;
  int* status;
  LookBuffer look;
};

// Four channels of one token, W neighbours at a time: as many as D, strides and alignment let be moved at once.
template <int W>
__device__ __forceinline__ int channel_of(int lane, int j) { return (j / W * kLanes + lane) * W + j % W; }

// What a thread has of a tile lies in shared memory, four channels of a token in a cell of its own, [step][thread]: nobody else reads
// or writes it, so nothing but the thread's own wait for its copies stands between them and their use.
template <int S, int WORDS> struct Cells {
  alignas(16) uint32_t w[S][kRunners][WORDS];      // (a copy's two ends lie on a boundary of its size)

  // Step s of this thread from p, its first channel of that token, where all channels of the strip exist ...
  template <int TY, int W>
  __device__ __forceinline__ void fetch(int s, const typename Elem<TY>::T* p) {
    constexpr int kBytes = W * elem_bytes(TY);
    if constexpr (kBytes >= 4) {
#pragma unroll
      for (int i = 0; i < kPer / W; ++i) copy<kBytes>(s, i, p + i * (kLanes * W), kBytes);
    }
  }
  // ... and where `room` channels do, from this thread's first on (0: no token); `base`: the tensor, an address that is good where nothing is
  // read.  (Two bytes are no asynchronous copy: load_all.)
  template <int TY, int W>
  __device__ __forceinline__ void fetch(int s, const typename Elem<TY>::T* p, const void* base, int room) {
    constexpr int kBytes = W * elem_bytes(TY);
    if constexpr (kBytes >= 4) {
#pragma unroll
      for (int i = 0; i < kPer / W; ++i) {
        const bool any = i * (kLanes * W) < room;
        copy<kBytes>(s, i, any ? p + i * (kLanes * W) : base, any ? kBytes : 0);
      }
    }
  }
  // All steps of a thread element by element, loads first.
  template <int TY, int W>
  __device__ __forceinline__ void load_all(const typename Elem<TY>::T* p, long long stride, int live, int room) {
    if constexpr (W * elem_bytes(TY) < 4) {
      Raw<TY, kPer> r[S];
#pragma unroll
      for (int s = 0; s < S; ++s) {
        r[s].zero();
#pragma unroll
        for (int j = 0; j < kPer; ++j)
          if (s < live && j * kLanes < room) raw_put(r[s], j, __ldg(p + s * stride + j * kLanes));
      }
#pragma unroll
      for (int s = 0; s < S; ++s) put(s, r[s]);
    }
  }
  template <int BYTES>
  __device__ __forceinline__ void copy(int s, int i, const void* from, int bytes) {      // (zeros beyond `bytes`)
    const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(&w[s][threadIdx.x][0])) + i * BYTES;
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(BYTES), "r"(bytes) : "memory");
  }
  template <int TY>
  __device__ __forceinline__ Raw<TY, kPer> take(int s) const {
    Raw<TY, kPer> r;
#pragma unroll
    for (int i = 0; i < Raw<TY, kPer>::kWords; ++i) r.w[i] = w[s][threadIdx.x][i];
    return r;
  }
  template <int TY>
  __device__ __forceinline__ void put(int s, const Raw<TY, kPer>& r) {
#pragma unroll
    for (int i = 0; i < Raw<TY, kPer>::kWords; ++i) w[s][threadIdx.x][i] = r.w[i];
  }
};
// p: this thread's first channel; room: channels from there on
template <int TY, int W>
__device__ __forceinline__ void store_token(const Raw<TY, kPer>& r, typename Elem<TY>::T* p, int room) {
  constexpr int kBytes = W * elem_bytes(TY), kWords = kBytes / 4;
#pragma unroll
  for (int i = 0; i < kPer / W; ++i) {
    if (i * (kLanes * W) >= room) continue;
    uint32_t* d = reinterpret_cast<uint32_t*>(p + i * (kLanes * W));
    if constexpr (kWords == 4) *reinterpret_cast<uint4*>(d) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    else if constexpr (kWords == 2) *reinterpret_cast<uint2*>(d) = make_uint2(r.w[i * 2], r.w[i * 2 + 1]);
    else if constexpr (kWords == 1) *d = r.w[i];
    else p[i * kLanes] = raw_take(r, i);
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
// What a tile hands on.  The state in front of a tile depends on all tiles before it; a tile leaves its own part, (sum of g,
// state from zero), in the work buffer as soon as it has it, 64 bits per channel, stored and loaded as one, so a word
// that is there is whole and needs no flag or fence beside it.  Unwritten words are all ones (the buffer is set so in front of the kernel).
//
// Three levels keep what a tile has to read at 15 words: the tiles of its group of 8 in front of it, the groups of its 8 groups in
// front of it (the last tile of a group leaves that word, from the group's words alone), and the state behind the 64 tiles before
// those (left by the last of them).  The order of the fold is that of the tokens whoever comes first.
//
// Tiles are taken by ticket, so a tile waits only for tiles whose CTAs run already and wait for earlier ones only.  Waits are
// bounded all the same: one that runs out leaves a code in the status word and lets everybody pass.
// ---------------------------------------------------------------------------------------------
constexpr int kFan = 8;
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

struct Ticket {
  int order, tile;               // of the tile in its sequence, as it is folded (from `tiles` on there is none) and from the first token on
  uint32_t seq;                  // sequence: strip of channels of a batch
  int room, live;                // channels of the strip, tokens of the tile
  long long state, record;       // where its strip begins in a state [B, D] and among the states that are kept
  long long x, g, d, h;          // its first element in x, g, d_h and in what is contiguous
};
template <int XT, int S> struct ForwardShared {
  struct Tile {
    Cells<S, elem_bytes(XT)> x;
    Cells<S, 4> c;                        // g, and over it the coefficients
  } tile[2];
  alignas(16) float2 part[2][kGroups][kChannels];      // per group of tokens: (sum of g, state from zero); the publisher puts the
                                                       // coefficient in the sum's place, the lookers the state in front of the group
  Ticket ticket[4];
};
template <int XT, int S> struct BackwardShared {
  struct Tile {
    Cells<S, elem_bytes(XT)> x, d;
    Cells<S, 4> c;
  } tile[2];
  alignas(16) float2 part[2][kGroups][kChannels];      // as above
  alignas(16) float back[2][kGroups][kChannels];       // the gradient that leaves a group towards earlier tokens, from zero; the lookers put that which comes into it
  Ticket ticket[4];
};
static_assert(2 * sizeof(ForwardShared<LETHE_BF16, forward_steps(LETHE_BF16)>) <= 230400 && 2 * sizeof(ForwardShared<LETHE_F32, forward_steps(LETHE_F32)>) <= 230400 &&
              2 * sizeof(BackwardShared<LETHE_BF16, backward_steps(LETHE_BF16)>) <= 230400 && 2 * sizeof(BackwardShared<LETHE_F32, backward_steps(LETHE_F32)>) <= 230400, "two CTAs on an SM");

// Where tile number `i` (in the order of the fold) of sequence `seq` stands among the three levels.
struct LookPlace {
  LookBuffer buf;
  long long group0, tile0;      // first words of its level: groups of its super, tiles of its group
  long long super;              // its super's word
  int n_groups, n_tiles;        // how many in front of it
  bool first_super, last;       // no tiles in front of its super; no tile behind it
  __device__ __forceinline__ bool closes_super() const { return n_tiles == kFan - 1 && n_groups == kFan - 1 && !last; }
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

// A looker: what comes in front of the tile in its channel; `first`: in front of the first tile.  The last tile of a group leaves the group's
// word.  A straight line where all words are there: one that does not exist is (0, 0), which is a step that changes nothing.
__device__ __forceinline__ float look_back(const LookPlace& p, int ch, float first, int* status) {
  const auto upper = [](unsigned long long v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); };
  const auto lower = [](unsigned long long v) { return __uint_as_float(static_cast<uint32_t>(v)); };
  constexpr int N = kFan - 1;
  const bool closes = p.n_tiles == N && !p.last;
  unsigned long long t[N], g[N], b = 0, own = 0;
  bool missing = false;
#pragma unroll
  for (int k = 0; k < N; ++k) t[k] = k < p.n_tiles ? look_load(p.at(0, p.tile0 + k, ch)) : 0;
#pragma unroll
  for (int k = 0; k < N; ++k) g[k] = k < p.n_groups ? look_load(p.at(1, p.group0 + k, ch)) : 0;
  if (!p.first_super) b = look_load(p.at(2, p.super - 1, ch));
  if (closes) own = look_load(p.at(0, p.tile0 + N, ch));
#pragma unroll
  for (int k = 0; k < N; ++k) missing = missing || t[k] == ~0ull;
  if (missing) {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (t[k] == ~0ull) t[k] = look_wait(p.at(0, p.tile0 + k, ch), p.buf.head, status);
  }
  float c[N];
#pragma unroll
  for (int k = 0; k < N; ++k) c[k] = decay_coef(lower(t[k]));
  if (closes) {
    if (own == ~0ull) own = look_wait(p.at(0, p.tile0 + N, ch), p.buf.head, status);
    float gs = 0.f, gh = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      gs += lower(t[k]);
      gh = decay_step(c[k], gh, upper(t[k]));
    }
    look_store(p.at(1, p.group0 + p.n_groups, ch), gs + lower(own), decay_step(decay_coef(lower(own)), gh, upper(own)));
  }
  missing = b == ~0ull;
#pragma unroll
  for (int k = 0; k < N; ++k) missing = missing || g[k] == ~0ull;
  if (missing) {
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (g[k] == ~0ull) g[k] = look_wait(p.at(1, p.group0 + k, ch), p.buf.head, status);
    if (b == ~0ull) b = look_wait(p.at(2, p.super - 1, ch), p.buf.head, status);
  }
  float carry = p.first_super ? first : upper(b);
#pragma unroll
  for (int k = 0; k < N; ++k) carry = decay_step(decay_coef(lower(g[k])), carry, upper(g[k]));
#pragma unroll
  for (int k = 0; k < N; ++k) carry = decay_step(c[k], carry, upper(t[k]));
  return carry;
}

// One thread takes tickets, and says for all what they stand for.
template <int S, bool BACK, bool PACK> struct TicketTaker {
  const DiagProblem& p;
  uint32_t have;      // the last one
  __device__ __forceinline__ void take() { have = p.tiles > 1 ? atomicAdd(p.look.head, 1u) + 1u : have + gridDim.x; }
  __device__ __forceinline__ Ticket named() const {
    Ticket t;
    t.order = static_cast<int>(have / p.seqs);
    t.tile = BACK ? p.tiles - 1 - t.order : t.order;
    t.seq = have - t.order * p.seqs;
    const long long b = PACK ? static_cast<long long>(t.seq) * p.pack : t.seq / static_cast<uint32_t>(p.strips);
    const long long ch0 = PACK ? 0 : (t.seq - b * p.strips) * kChannels, t0 = static_cast<long long>(t.tile) * (kGroups * S);
    const long long there = PACK ? (p.B - b < p.pack ? p.B - b : p.pack) * p.D : p.D - ch0;
    t.room = static_cast<int>(there < kChannels ? there : kChannels);
    t.live = static_cast<int>(p.L - t0 < kGroups * S ? p.L - t0 : kGroups * S);
    t.state = b * p.D + ch0;
    t.record = (b * p.records + (BACK ? t.tile : 2 * t.tile)) * p.D + ch0;
    t.x = b * p.x_batch + t0 * p.x_token + ch0;
    t.g = b * p.g_batch + t0 * p.g_token + ch0;
    t.d = b * p.d_batch + t0 * p.d_token + ch0;
    t.h = (b * p.L + t0) * p.D + ch0;
    return t;
  }
};
// Where channel `ch` of a strip lies, from the strip's first one on, in a tensor with a stride between batches.
template <bool PACK>
__device__ __forceinline__ long long channel_place(const DiagProblem& p, int ch, long long batch) {
  if constexpr (!PACK) return ch;
  const int D = static_cast<int>(p.D);
  return ch / D * batch + ch % D;
}
// This thread's first element of a tensor, in a tile whose first element is the tensor's.
template <int TY>
__device__ __forceinline__ typename Elem<TY>::T* own_part(const void* tensor, long long token, int first_token, long long place) {
  return static_cast<typename Elem<TY>::T*>(const_cast<void*>(tensor)) + first_token * token + place;
}

// Barriers from one role to the next, two of each for even and odd tiles: a tile's parts are there (runners to publisher), its word has
// gone out (publisher to lookers), its starts are there (lookers to runners).
constexpr int kBarParts = 1, kBarOut = 3, kBarStarts = 5;
template <int N> __device__ __forceinline__ void bar_sync(int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory"); }
template <int N> __device__ __forceinline__ void bar_arrive(int id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(N) : "memory"); }
constexpr int kPartsThreads = kRunners + kChannels, kOutThreads = 2 * kChannels, kStartsThreads = kChannels + kRunners;

// The CTAs take tiles until there are none; a CTA's tickets ascend, and it takes tickets ahead: the tile of the lowest ticket that is not
// done is one that its CTA has begun or begins next, so somebody always can go on.
//
// Runners go over a tile's tokens twice, and over those of the next tile the first time before they go over this one the second time.
// Publishers fold a tile's parts and let its word go out, lookers wait for the words of others.  So a tile's word waits for nobody,
// and looking back has the time of a run.  Steps on the way (B1 L65536 D2048 bf16, forward / backward in us): tiles in registers, two CTAs on
// an SM, 462 / 651; the next tile by asynchronous copies and fewer operations 344 / 462; folding and looking in warps of their own,
// a word behind the looking of the tile before it, 299 / 700; as it is 239 / 475; two channels by one instruction and the places of a
// tile worked out once 226 / 425.  Tried beside 239 / 475 and left (not measured again since): whole tiles by tensor-map copies 240 / 490, four small CTAs without roles 627 / 569, one
// more ticket ahead 255 / 506, tiles fetched to L2 row by row 388 / 638, tickets dealt out beforehand in a cooperative launch 228 / 470
// (B2 L2048 D1024 14.5 + 21.1 against 15.6 + 23).
template <int XT, int GT, int WIDTH, bool COMP>
__global__ void __launch_bounds__(kScanThreads, 2) diag_forward_kernel(const DiagProblem p) {
  constexpr bool PACK = WIDTH == kPacked;
  constexpr int W = PACK ? kPer : WIDTH;
  using X = typename Elem<XT>::T;
  constexpr int S = forward_steps(XT);
  extern __shared__ __align__(16) unsigned char smem[];
  auto& sh = *reinterpret_cast<ForwardShared<XT, S>*>(smem);
  TicketTaker<S, false, PACK> tickets{p, blockIdx.x - gridDim.x};
  const bool taker = threadIdx.x == kPublisher;
  if (taker) {
    tickets.take();
    sh.ticket[0] = tickets.named();
    tickets.take();
    sh.ticket[1] = tickets.named();
  }
  __syncthreads();
  if (threadIdx.x >= kLooker) {
    const int ch = threadIdx.x - kLooker;
    const long long record_of = channel_place<PACK>(p, ch, p.records * p.D);
    for (int n = 0;; ++n) {
      const Ticket cur = sh.ticket[n & 3];
      if (cur.order >= p.tiles) break;
      const LookPlace look(p.look, cur.seq, p.tiles, cur.order);
      auto& part = sh.part[n & 1];
      const long long state_at = cur.state + ch;
      float carry = ch < cur.room && p.h0 ? p.h0[state_at] : 0.f;
      bar_sync<kOutThreads>(kBarOut + (n & 1));
      if (p.tiles > 1) carry = look_back(look, ch, carry, p.status);
      const float entry = carry;
      float middle = 0.f;
      float2 own[kGroups];
#pragma unroll
      for (int i = 0; i < kGroups; ++i) own[i] = part[i][ch];
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        if (i == kGroups / 2) middle = carry;
        part[i][ch].x = carry;
        carry = decay_step(own[i].x, carry, own[i].y);
      }
      bar_arrive<kStartsThreads>(kBarStarts + (n & 1));
      if (p.tiles > 1 && look.closes_super()) look_store(look.at(2, look.super, ch), 0.f, carry);
      if (p.states && ch < cur.room) {
        float* to = p.states + cur.record + record_of;
        to[0] = entry;
        if (2 * cur.tile + 1 < p.records) to[p.D] = middle;
      }
      if (p.hT && ch < cur.room && cur.tile == p.tiles - 1) p.hT[state_at] = carry;
    }
    return;
  }
  if (threadIdx.x >= kPublisher) {
    const int ch = threadIdx.x - kPublisher;
    for (int n = 0;; ++n) {
      const Ticket cur = sh.ticket[n & 3];
      if (cur.order >= p.tiles) break;
      const LookPlace look(p.look, cur.seq, p.tiles, cur.order);
      auto& part = sh.part[n & 1];
      bar_sync<kPartsThreads>(kBarParts + (n & 1));
      if (taker) tickets.take();
      float ts = 0.f, th = 0.f;
      float2 v[kGroups];
#pragma unroll
      for (int i = 0; i < kGroups; ++i) v[i] = part[i][ch];
#pragma unroll
      for (int i = 0; i < kGroups; i += 2) {
        ts += v[i].x;
        ts += v[i + 1].x;
        decay_coefs(v[i].x, v[i + 1].x);
      }
#pragma unroll
      for (int i = 0; i < kGroups; ++i) th = decay_step(v[i].x, th, v[i].y);
      if (p.tiles > 1 && !look.last) look_store(look.at(0, look.tile0 + look.n_tiles, ch), ts, th);
#pragma unroll
      for (int i = 0; i < kGroups; ++i) part[i][ch].x = v[i].x;
      if (taker) sh.ticket[(n + 2) & 3] = tickets.named();
      bar_arrive<kOutThreads>(kBarOut + (n & 1));
    }
    return;
  }
  const int lane = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  using GE = typename Elem<GT>::T;
  const X* const x0 = own_part<XT>(p.x, p.x_token, grp * S, channel_place<PACK>(p, lane * W, p.x_batch));
  const GE* const g0 = own_part<GT>(p.g, p.g_token, grp * S, channel_place<PACK>(p, lane * W, p.g_batch));
  X* const h0 = own_part<XT>(p.h, p.D, grp * S, channel_place<PACK>(p, lane * W, p.L * p.D));
  const auto fetch = [&](const Ticket& t, int slot) {
    if (t.order < p.tiles) {
      auto& tile = sh.tile[slot];
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int room = s < t.live - grp * S ? t.room - lane * W : 0;
        tile.x.template fetch<XT, W>(s, x0 + t.x + s * p.x_token, p.x, room);
        tile.c.template fetch<GT, W>(s, g0 + t.g + s * p.g_token, p.g, room);
      }
      tile.x.template load_all<XT, W>(x0 + t.x, p.x_token, t.live - grp * S, t.room - lane * W);
      tile.c.template load_all<GT, W>(g0 + t.g, p.g_token, t.live - grp * S, t.room - lane * W);
    }
    commit();
  };
  const auto first_run = [&](int slot) {
    auto& tile = sh.tile[slot];
    float sum[kPer], st[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum[j] = st[j] = 0.f;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const auto gr = tile.c.template take<GT>(s);
      const auto xr = tile.x.template take<XT>(s);
      Raw<LETHE_F32, kPer> cr;
#pragma unroll
      for (int j = 0; j < kPer; j += 2) {
        const float a0 = gr.get(j), a1 = gr.get(j + 1);
        float c0 = a0, c1 = a1;
        decay_coefs(c0, c1);
        cr.set2(j, c0, c1);
        add_to(sum[j], sum[j + 1], a0, a1);
        const float v0 = xr.get(j), v1 = xr.get(j + 1);
        decay_steps(c0, c1, by_diff(a0), by_diff(a1), st[j], st[j + 1], COMP ? v0 * forgotten(c0) : v0, COMP ? v1 * forgotten(c1) : v1);
      }
      tile.c.put(s, cr);
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) sh.part[slot][grp][channel_of<W>(lane, j)] = make_float2(sum[j], st[j]);
    bar_arrive<kPartsThreads>(kBarParts + slot);
  };
  fetch(sh.ticket[0], 0);
  fetch(sh.ticket[1], 1);
  if (sh.ticket[0].order < p.tiles) {
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    first_run(0);
  }
  for (int n = 0;; ++n) {
    const Ticket& cur = sh.ticket[n & 3];
    if (cur.order >= p.tiles) break;
    const int slot = n & 1;
    if (sh.ticket[(n + 1) & 3].order < p.tiles) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      first_run(slot ^ 1);
    }
    auto& tile = sh.tile[slot];
    X* h = h0 + cur.h;
    const int live = cur.live - grp * S, room = cur.room - lane * W;
    const bool whole = live >= S && cur.room == kChannels;
    float st[kPer];
    bar_sync<kStartsThreads>(kBarStarts + slot);
#pragma unroll
    for (int j = 0; j < kPer; ++j) st[j] = sh.part[slot][grp][channel_of<W>(lane, j)].x;
    // a cell that has been read takes its step of the tile after the next
    const Ticket& after = sh.ticket[(n + 2) & 3];
    const X* xn = x0 + after.x;
    const GE* gn = g0 + after.g;
    const bool more = after.order < p.tiles;
    const int live_n = after.live - grp * S, room_n = after.room - lane * W;
    const bool whole_n = more && live_n >= S && after.room == kChannels;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const auto xr = tile.x.template take<XT>(s);
      const auto cr = tile.c.template take<LETHE_F32>(s);
      if (whole_n) {
        tile.x.template fetch<XT, W>(s, xn);
        tile.c.template fetch<GT, W>(s, gn);
      } else if (more) {
        tile.x.template fetch<XT, W>(s, xn, p.x, s < live_n ? room_n : 0);
        tile.c.template fetch<GT, W>(s, gn, p.g, s < live_n ? room_n : 0);
      }
      xn += p.x_token;
      gn += p.g_token;
#pragma unroll
      for (int j = 0; j < kPer; j += 2) {
        const float c0 = cr.get(j), c1 = cr.get(j + 1), v0 = xr.get(j), v1 = xr.get(j + 1);
        decay_steps(c0, c1, is_diff(c0), is_diff(c1), st[j], st[j + 1], COMP ? v0 * forgotten(c0) : v0, COMP ? v1 * forgotten(c1) : v1);
      }
      if (whole) store_token<XT, W>(packed<XT>(st), h, kChannels);
      else if (s < live) store_token<XT, W>(packed<XT>(st), h, room);
      h += p.D;
    }
    if (more) {
      tile.x.template load_all<XT, W>(x0 + after.x, p.x_token, live_n, room_n);
      tile.c.template load_all<GT, W>(g0 + after.g, p.g_token, live_n, room_n);
    }
    commit();
  }
}

template <int XT, int GT, int WIDTH, bool COMP>
__global__ void __launch_bounds__(kScanThreads, 2) diag_backward_kernel(const DiagProblem p) {
  constexpr bool PACK = WIDTH == kPacked;
  constexpr int W = PACK ? kPer : WIDTH;
  using X = typename Elem<XT>::T;
  using G = typename Elem<GT>::T;
  constexpr int S = backward_steps(XT);
  extern __shared__ __align__(16) unsigned char smem[];
  auto& sh = *reinterpret_cast<BackwardShared<XT, S>*>(smem);
  TicketTaker<S, true, PACK> tickets{p, blockIdx.x - gridDim.x};
  const bool taker = threadIdx.x == kPublisher;
  if (taker) {
    tickets.take();
    sh.ticket[0] = tickets.named();
    tickets.take();
    sh.ticket[1] = tickets.named();
  }
  __syncthreads();
  if (threadIdx.x >= kLooker) {
    const int ch = threadIdx.x - kLooker;
    const long long record_of = channel_place<PACK>(p, ch, p.records * p.D);
    for (int n = 0;; ++n) {
      const Ticket cur = sh.ticket[n & 3];
      if (cur.order >= p.tiles) break;
      const LookPlace look(p.look, cur.seq, p.tiles, cur.order);
      auto& part = sh.part[n & 1];
      auto& back = sh.back[n & 1];
      const long long state_at = cur.state + ch;
      float carry = ch < cur.room && p.dhT ? p.dhT[state_at] : 0.f;
      float st = ch < cur.room ? p.states[cur.record + record_of] : 0.f;
      bar_sync<kOutThreads>(kBarOut + (n & 1));
      if (p.tiles > 1) carry = look_back(look, ch, carry, p.status);
      float2 own[kGroups];
      float e[kGroups];
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        own[i] = part[i][ch];
        e[i] = back[i][ch];
      }
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {      // (two chains, one from each end)
        const int k = kGroups - 1 - i;
        back[k][ch] = carry;
        carry = decay_step(own[k].x, carry, e[k]);
        part[i][ch].x = st;
        st = decay_step(own[i].x, st, own[i].y);
      }
      bar_arrive<kStartsThreads>(kBarStarts + (n & 1));
      if (p.tiles > 1 && look.closes_super()) look_store(look.at(2, look.super, ch), 0.f, carry);
      if (p.dh0 && ch < cur.room && cur.tile == 0) p.dh0[state_at] = carry;
    }
    return;
  }
  if (threadIdx.x >= kPublisher) {
    const int ch = threadIdx.x - kPublisher;
    for (int n = 0;; ++n) {
      const Ticket cur = sh.ticket[n & 3];
      if (cur.order >= p.tiles) break;
      const LookPlace look(p.look, cur.seq, p.tiles, cur.order);
      auto& part = sh.part[n & 1];
      bar_sync<kPartsThreads>(kBarParts + (n & 1));
      if (taker) tickets.take();
      float ts = 0.f, te = 0.f, c[kGroups], e[kGroups];
#pragma unroll
      for (int i = 0; i < kGroups; ++i) {
        c[i] = part[i][ch].x;
        e[i] = sh.back[n & 1][i][ch];
      }
#pragma unroll
      for (int i = 0; i < kGroups; i += 2) {
        ts += c[i];
        ts += c[i + 1];
        decay_coefs(c[i], c[i + 1]);
      }
#pragma unroll
      for (int i = kGroups - 1; i >= 0; --i) te = decay_step(c[i], te, e[i]);
      if (p.tiles > 1 && !look.last) look_store(look.at(0, look.tile0 + look.n_tiles, ch), ts, te);
#pragma unroll
      for (int i = 0; i < kGroups; ++i) part[i][ch].x = c[i];
      if (taker) sh.ticket[(n + 2) & 3] = tickets.named();
      bar_arrive<kOutThreads>(kBarOut + (n & 1));
    }
    return;
  }
  const int lane = threadIdx.x % kLanes, grp = threadIdx.x / kLanes;
  const auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
  using GE = typename Elem<GT>::T;
  const X* const x0 = own_part<XT>(p.x, p.x_token, grp * S, channel_place<PACK>(p, lane * W, p.x_batch));
  const GE* const g0 = own_part<GT>(p.g, p.g_token, grp * S, channel_place<PACK>(p, lane * W, p.g_batch));
  const X* const d0 = own_part<XT>(p.d_h, p.d_token, grp * S, channel_place<PACK>(p, lane * W, p.d_batch));
  X* const dx0 = own_part<XT>(p.dx, p.D, grp * S, channel_place<PACK>(p, lane * W, p.L * p.D));
  G* const dg0 = own_part<GT>(p.dg, p.D, grp * S, channel_place<PACK>(p, lane * W, p.L * p.D));
  const auto fetch = [&](const Ticket& t, int slot) {
    if (t.order < p.tiles) {
      auto& tile = sh.tile[slot];
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int room = s < t.live - grp * S ? t.room - lane * W : 0;
        tile.x.template fetch<XT, W>(s, x0 + t.x + s * p.x_token, p.x, room);
        tile.c.template fetch<GT, W>(s, g0 + t.g + s * p.g_token, p.g, room);
        if (p.d_h) tile.d.template fetch<XT, W>(s, d0 + t.d + s * p.d_token, p.d_h, room);
      }
      tile.x.template load_all<XT, W>(x0 + t.x, p.x_token, t.live - grp * S, t.room - lane * W);
      tile.c.template load_all<GT, W>(g0 + t.g, p.g_token, t.live - grp * S, t.room - lane * W);
      if (p.d_h) tile.d.template load_all<XT, W>(d0 + t.d, p.d_token, t.live - grp * S, t.room - lane * W);
    }
    commit();
  };
  const auto first_run = [&](int slot) {
    auto& tile = sh.tile[slot];
    float c[S][kPer], sum[kPer], st[kPer], e[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum[j] = st[j] = e[j] = 0.f;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const auto gr = tile.c.template take<GT>(s);
      const auto xr = tile.x.template take<XT>(s);
      Raw<LETHE_F32, kPer> cr;
#pragma unroll
      for (int j = 0; j < kPer; j += 2) {
        const float a0 = gr.get(j), a1 = gr.get(j + 1);
        float c0 = a0, c1 = a1;
        decay_coefs(c0, c1);
        cr.set2(j, c0, c1);
        c[s][j] = c0;
        c[s][j + 1] = c1;
        add_to(sum[j], sum[j + 1], a0, a1);
        const float v0 = xr.get(j), v1 = xr.get(j + 1);
        decay_steps(c0, c1, by_diff(a0), by_diff(a1), st[j], st[j + 1], COMP ? v0 * forgotten(c0) : v0, COMP ? v1 * forgotten(c1) : v1);
      }
      tile.c.put(s, cr);
    }
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
      const auto dr = tile.d.template take<XT>(s);
#pragma unroll
      for (int j = 0; j < kPer; j += 2) {
        add_to(e[j], e[j + 1], dr.get(j), dr.get(j + 1));
        decay_over(c[s][j], c[s][j + 1], e[j], e[j + 1]);
      }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int ch = channel_of<W>(lane, j);
      sh.part[slot][grp][ch] = make_float2(sum[j], st[j]);
      sh.back[slot][grp][ch] = e[j];
    }
    bar_arrive<kPartsThreads>(kBarParts + slot);
  };
  if (!p.d_h) {      // no gradient of h: zeros, for good
    Raw<XT, kPer> none;
    none.zero();
#pragma unroll
    for (int s = 0; s < S; ++s) {
      sh.tile[0].d.put(s, none);
      sh.tile[1].d.put(s, none);
    }
  }
  fetch(sh.ticket[0], 0);
  fetch(sh.ticket[1], 1);
  if (sh.ticket[0].order < p.tiles) {
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    first_run(0);
  }
  for (int n = 0;; ++n) {
    const Ticket& cur = sh.ticket[n & 3];
    if (cur.order >= p.tiles) break;
    const int slot = n & 1;
    if (sh.ticket[(n + 1) & 3].order < p.tiles) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      first_run(slot ^ 1);
    }
    auto& tile = sh.tile[slot];
    const int live = cur.live - grp * S, room = cur.room - lane * W;
    const bool whole = live >= S && cur.room == kChannels && p.dx && p.dg;
    float before[S][kPer], c[S][kPer], st[kPer], e[kPer];
    bar_sync<kStartsThreads>(kBarStarts + slot);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int ch = channel_of<W>(lane, j);
      st[j] = sh.part[slot][grp][ch].x;
      e[j] = sh.back[slot][grp][ch];
    }
    const Ticket& after = sh.ticket[(n + 2) & 3];
    const X* xn = x0 + after.x;
    const GE* gn = g0 + after.g;
    const bool more = after.order < p.tiles;
    const int live_n = after.live - grp * S, room_n = after.room - lane * W;
    const bool whole_n = more && live_n >= S && after.room == kChannels && p.d_h;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const auto xr = tile.x.template take<XT>(s);
      const auto cr = tile.c.template take<LETHE_F32>(s);
      if (whole_n) {
        tile.x.template fetch<XT, W>(s, xn);
        tile.c.template fetch<GT, W>(s, gn);
      } else if (more) {
        tile.x.template fetch<XT, W>(s, xn, p.x, s < live_n ? room_n : 0);
        tile.c.template fetch<GT, W>(s, gn, p.g, s < live_n ? room_n : 0);
      }
      xn += p.x_token;
      gn += p.g_token;
#pragma unroll
      for (int j = 0; j < kPer; j += 2) {
        const float c0 = cr.get(j), c1 = cr.get(j + 1), v0 = xr.get(j), v1 = xr.get(j + 1);
        c[s][j] = c0;
        c[s][j + 1] = c1;
        before[s][j] = COMP ? st[j] - v0 : st[j];
        before[s][j + 1] = COMP ? st[j + 1] - v1 : st[j + 1];
        decay_steps(c0, c1, is_diff(c0), is_diff(c1), st[j], st[j + 1], COMP ? v0 * forgotten(c0) : v0, COMP ? v1 * forgotten(c1) : v1);
      }
    }
    const X* dn = d0 + after.d + (S - 1) * p.d_token;
    X* dx = dx0 + cur.h + (S - 1) * p.D;
    G* dg = dg0 + cur.h + (S - 1) * p.D;
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
      const auto dr = tile.d.template take<XT>(s);
      if (whole_n) tile.d.template fetch<XT, W>(s, dn);
      else if (more && p.d_h) tile.d.template fetch<XT, W>(s, dn, p.d_h, s < live_n ? room_n : 0);
      dn -= p.d_token;
      float vx[kPer], vg[kPer];
#pragma unroll
      for (int j = 0; j < kPer; j += 2) {
        add_to(e[j], e[j + 1], dr.get(j), dr.get(j + 1));
        vx[j] = COMP ? e[j] * forgotten(c[s][j]) : e[j];
        vx[j + 1] = COMP ? e[j + 1] * forgotten(c[s][j + 1]) : e[j + 1];
        decay_over(c[s][j], c[s][j + 1], e[j], e[j + 1]);
        const F2 v = f2(e[j], e[j + 1]) * f2(before[s][j], before[s][j + 1]);
        vg[j] = lo(v);
        vg[j + 1] = hi(v);
      }
      if (whole) {
        store_token<XT, W>(packed<XT>(vx), dx, kChannels);
        store_token<GT, W>(packed<GT>(vg), dg, kChannels);
      } else if (s < live) {
        if (p.dx) store_token<XT, W>(packed<XT>(vx), dx, room);
        if (p.dg) store_token<GT, W>(packed<GT>(vg), dg, room);
      }
      dx -= p.D;
      dg -= p.D;
    }
    if (more) {
      tile.x.template load_all<XT, W>(x0 + after.x, p.x_token, live_n, room_n);
      tile.c.template load_all<GT, W>(g0 + after.g, p.g_token, live_n, room_n);
      if (p.d_h) tile.d.template load_all<XT, W>(d0 + after.d, p.d_token, live_n, room_n);
    }
    commit();
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
    if (w == kPacked) return last(std::integral_constant<int, kPacked>());
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

static long long tiles_of(long long L, int xt, bool backward) {
  const int n = kGroups * (backward ? backward_steps(xt) : forward_steps(xt));
  return (L - 1) / n + 1;      // (L + n - 1 need not fit)
}
static long long strips_of(long long D) { return (D - 1) / kChannels + 1; }
// tiles and what they hand on are counted in 32 bits
static bool countable(long long B, long long strips, long long tiles) {
  return strips <= INT32_MAX && B <= INT32_MAX / strips && tiles <= INT32_MAX / (B * strips);
}
static int diag_problem(const LetheGdnDiagArgs* a, DiagProblem* p, bool backward) {
  if (!a) return kErrNull;
  if (a->B <= 0 || a->L <= 0 || a->D <= 0 || !types_ok(a->x_type, a->g_type)) return kErrDims;
  if (!a->x || !a->g || !a->status || (!backward && !a->h) || (backward && !a->states)) return kErrNull;
  const long long tiles = tiles_of(a->L, a->x_type, backward), strips = strips_of(a->D);
  if (!countable(a->B, strips, tiles)) return kErrDims;
  if (!on_elements(a->x_type, a->x, a->h, a->d_h, a->dx) || !on_elements(a->g_type, a->g, a->dg) ||
      !on_elements(LETHE_F32, a->h0, a->hT, a->states, a->dhT, a->dh0, a->status)) return kErrAlign;
  *p = {a->B, a->L, a->D, a->x, a->x_batch, a->x_token, a->g, a->g_batch, a->g_token, a->h0, a->h, a->hT, a->states, a->d_h, a->d_h_batch,
        a->d_h_token, a->dhT, a->dx, a->dg, a->dh0, static_cast<int>(tiles), static_cast<int>(strips), tiles_of(a->L, a->x_type, true),
        static_cast<uint32_t>(a->B * strips), 1, 0, a->status, {}};
  if (tiles > 1) {
    if (!a->work) return kErrNull;
    if (reinterpret_cast<uintptr_t>(a->work) & 15) return kErrAlign;
    const LookSizes n = look_sizes(p->seqs, tiles);
    if (a->work_bytes < n.bytes()) return kErrWorkspace;
    p->look_bytes = n.bytes();
    p->look.head = static_cast<uint32_t*>(a->work);
    p->look.word[0] = reinterpret_cast<unsigned long long*>(static_cast<char*>(a->work) + kLookHead);
    for (int i = 1; i < 3; ++i) p->look.word[i] = p->look.word[i - 1] + n.count[i - 1] * kChannels;
  }
  return kOk;
}
// elements that can be moved at once
template <typename F>
static int widest(F&& fits) { return fits(4) ? 4 : fits(2) ? 2 : 1; }

// Few channels: a strip of 64 takes those of as many batches as fit (bf16, forward + backward in us, one batch / as many: 64 x 16384 x 8
// 104 + 191 / 39 + 56, 16 x 16384 x 32 37 + 62 / 27 + 42).  A kernel of its own: with the places of a channel open at run time the others
// spill more (B1 L65536 D2048 backward 424 / 442).  The work buffer is that of a strip for each batch, all of it cleared.
static int pack_batches(DiagProblem* p, int w) {
  if (w != kPer || p->D > kChannels / 2 || p->B < 2) return w;
  p->pack = static_cast<int>(kChannels / p->D);
  p->seqs = static_cast<uint32_t>((p->B + p->pack - 1) / p->pack);
  return kPacked;
}

template <typename Shared>
static int launch_scan_tiles(void (*kern)(DiagProblem), const DiagProblem& p, SmemAttr& attr, cudaStream_t st) {
  if (int e = attr.set(kern, sizeof(Shared))) return e;
  // all ones: no word is there yet, and the ticket before the first
  if (p.tiles > 1 && cudaMemsetAsync(p.look.head, 0xff, p.look_bytes, st) != cudaSuccess) return kErrLaunch;
  const uint32_t total = p.seqs * static_cast<uint32_t>(p.tiles), room = static_cast<uint32_t>(2 * sm_count());
  kern<<<total < room ? total : room, kScanThreads, sizeof(Shared), st>>>(p);
  return launched();
}

}  // namespace lg

extern "C" size_t lethe_gdn_diag_states_bytes(int64_t B, int64_t L, int64_t D, int32_t x_type) {
  using namespace lg;
  if (B <= 0 || L <= 0 || D <= 0 || !types_ok(x_type, LETHE_F32)) return 0;
  return static_cast<size_t>(B) * tiles_of(L, x_type, true) * D * sizeof(float);
}
extern "C" size_t lethe_gdn_diag_work_bytes(int64_t B, int64_t L, int64_t D, int32_t x_type, int32_t backward) {
  using namespace lg;
  if (B <= 0 || L <= 0 || D <= 0 || !types_ok(x_type, LETHE_F32)) return 0;
  const long long tiles = tiles_of(L, x_type, backward != 0), strips = strips_of(D);
  return tiles > 1 && countable(B, strips, tiles) ? look_sizes(B * strips, tiles).bytes() : 0;      // (0 too where the call itself refuses)
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
  const int width = pack_batches(&p, w);
  return by_type(a->x_type, a->g_type, width, a->complement != 0, [&](auto x, auto g, auto n, auto c) {
    static SmemAttr attr;
    return launch_scan_tiles<ForwardShared<x.value, forward_steps(x.value)>>(diag_forward_kernel<x.value, g.value, n.value, c.value>, p, attr, static_cast<cudaStream_t>(stream));
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
  const int width = pack_batches(&p, w);
  return by_type(a->x_type, a->g_type, width, a->complement != 0, [&](auto x, auto g, auto n, auto c) {
    static SmemAttr attr;
    return launch_scan_tiles<BackwardShared<x.value, backward_steps(x.value)>>(diag_backward_kernel<x.value, g.value, n.value, c.value>, p, attr, static_cast<cudaStream_t>(stream));
  });
}

extern "C" int lethe_gdn_diag_step(const LetheGdnDiagArgs* a, float* state, void* stream) {
  using namespace lg;
  if (!a) return kErrNull;
  if (a->B <= 0 || a->D <= 0 || !types_ok(a->x_type, a->g_type)) return kErrDims;
  if (!a->x || !a->g || !a->h || !state) return kErrNull;
  if (!on_elements(a->x_type, a->x, a->h) || !on_elements(a->g_type, a->g) || !on_elements(LETHE_F32, state)) return kErrAlign;
  const bool vec = a->D % kPer == 0 && on_boundary(a->x, a->x_type, kPer, a->x_batch) && on_boundary(a->g, a->g_type, kPer, a->g_batch) &&
                   on_boundary(a->h, a->x_type, kPer) && on_boundary(state, LETHE_F32, kPer);
  const long long blocks = (a->D - 1) / (256 * (vec ? kPer : 1)) + 1;
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
