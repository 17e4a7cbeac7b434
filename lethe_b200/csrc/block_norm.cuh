// Rows of the norms in front of and behind a block: who holds what of a row, row sums, column sums over rows.
//
// A row of D values is held by T threads with R pieces of 8 values each (T R 8 >= D) and stays in registers from its loads to its
// stores; a CTA has one row at a time, or as many as fill 256 threads.  Sums over up to a warp are butterflies, beyond that the warps of a
// row meet in shared memory.  CTAs go over the rows with the grid's stride, so that what belongs to a column (weights, sums for their
// gradients) stays in registers as well, and the next rows are under way by asynchronous copies (RowRing): with loads at the head of
// each turn instead, residual_norm of 16384 x 4096 bf16 took 132 us forward and 267 backward, against 92 and 167 with the ring alone.
// Sums over rows: a CTA's share in the order of its rows, the CTAs' shares by a kernel of its own in the order of the CTAs.  No
// atomics: two runs give the same bits.
#pragma once
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "elem.cuh"
#include "host_util.h"

namespace lg {

constexpr int kNormMaxD = 8192;

// CTAs of a backward at most: what the work buffer holds partial sums of
inline int norm_parts_max(int D) { return D <= 2048 ? 1024 : 320; }

// W: neighbours that are moved at once: 16 bytes of the widest type (8 or 4 values) where D, strides and boundaries allow it, else fewer.  With
// 8 values of fp32, in two moves, every move of a warp would take half of each sector it touches.
template <int T_, int R_, int W_>
struct RowShape {
  static constexpr int T = T_, R = R_, N = R_ * 8, P = N / 2;      // values and pairs of a thread
  static constexpr int W = W_, kMoves = N / W;
  static constexpr int kThreads = T > 256 ? T : 256, kRows = kThreads / T;
  static constexpr int kWarps = kThreads / 32;
  static constexpr int kColumnBytes = kRows > 1 ? kThreads * N * 4 : 0;      // what column_share wants
  // column of value n (of N) that thread t of a row holds
  __device__ __forceinline__ static int col(int t, int n) { return (n / W * T + t) * W + n % W; }

  template <int TY>
  __device__ __forceinline__ static void load(Raw<TY, 8> (&r)[R], const void* row, int t, int D) {
    const typename Elem<TY>::T* p = static_cast<const typename Elem<TY>::T*>(row);
#pragma unroll
    for (int i = 0; i < R; ++i) r[i].zero();
#pragma unroll
    for (int m = 0; m < kMoves; ++m) {
      const int c = col(t, m * W);
      if (c >= D) continue;
      constexpr int kWords = W * elem_bytes(TY) / 4;
      if constexpr (kWords == 0) {
        raw_put(r[m / 8], m % 8, __ldg(p + c));
      } else {
        uint32_t* to = &r[m * W / 8].w[m * W % 8 * elem_bytes(TY) / 4];
        const uint32_t* from = reinterpret_cast<const uint32_t*>(p + c);
        if constexpr (kWords == 1) to[0] = __ldg(from);
        else if constexpr (kWords == 2) {
          const uint2 v = __ldg(reinterpret_cast<const uint2*>(from));
          to[0] = v.x;
          to[1] = v.y;
        } else {
#pragma unroll
          for (int k = 0; k < kWords; k += 4) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(from + k));
            to[k] = v.x;
            to[k + 1] = v.y;
            to[k + 2] = v.z;
            to[k + 3] = v.w;
          }
        }
      }
    }
  }
  template <int TY>
  __device__ __forceinline__ static void store(const Raw<TY, 8> (&r)[R], void* row, int t, int D) {
    typename Elem<TY>::T* p = static_cast<typename Elem<TY>::T*>(row);
#pragma unroll
    for (int m = 0; m < kMoves; ++m) {
      const int c = col(t, m * W);
      if (c >= D) continue;
      constexpr int kWords = W * elem_bytes(TY) / 4;
      if constexpr (kWords == 0) {
        p[c] = raw_take(r[m / 8], m % 8);
      } else {
        const uint32_t* from = &r[m * W / 8].w[m * W % 8 * elem_bytes(TY) / 4];
        uint32_t* to = reinterpret_cast<uint32_t*>(p + c);
        if constexpr (kWords == 1) to[0] = from[0];
        else if constexpr (kWords == 2) *reinterpret_cast<uint2*>(to) = make_uint2(from[0], from[1]);
        else
#pragma unroll
          for (int k = 0; k < kWords; k += 4) *reinterpret_cast<uint4*>(to + k) = make_uint4(from[k], from[k + 1], from[k + 2], from[k + 3]);
      }
    }
  }
  template <int TY>
  __device__ __forceinline__ static void store(const F2 (&v)[P], void* row, int t, int D) {
    Raw<TY, 8> r[R];
#pragma unroll
    for (int n = 0; n < P; ++n) r[n / 4].set2(n % 4, v[n]);
    store<TY>(r, row, t, D);
  }
  // a vector of D values (weight, scale), fp32 or XT; `none` where there is no vector
  template <int XT>
  __device__ __forceinline__ static void vector(F2 (&v)[P], const void* p, bool f32, int t, int D, float none) {
    const auto one = [&](int n) {
      const int c = col(t, n);
      if (!p || c >= D) return none;
      return f32 ? __ldg(static_cast<const float*>(p) + c) : to_f32(__ldg(static_cast<const typename Elem<XT>::T*>(p) + c));
    };
#pragma unroll
    for (int n = 0; n < P; ++n) v[n] = f2(one(2 * n), one(2 * n + 1));
  }
  // sums of K values over the threads of a row, in all of them.  `buf`: this sum's place in shared memory, not that of the sum before.
  template <int K>
  __device__ __forceinline__ static void row_sums(float (&s)[K], float (*buf)[kWarps]) {
#pragma unroll
    for (int m = (T < 32 ? T : 32) / 2; m >= 1; m >>= 1)
#pragma unroll
      for (int k = 0; k < K; ++k) s[k] += __shfl_xor_sync(0xffffffffu, s[k], m);
    if constexpr (T > 32) {
      constexpr int kOfRow = T / 32;
      const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
      if (lane == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) buf[k][warp] = s[k];
      __syncthreads();
      // one sum: every thread adds what the warps left, four chains of it; several: each lane one warp's, and butterflies (16384 x 4096 bf16
      // in us, added / butterflies: forward, sums one by one, 96 / 103; backward, three together, 161 / 150)
      if constexpr (K == 1 && kOfRow >= 4) {
        const float4* p = reinterpret_cast<const float4*>(&buf[0][warp / kOfRow * kOfRow]);
        float4 a = p[0];
#pragma unroll
        for (int i = 1; i < kOfRow / 4; ++i) {
          const float4 c = p[i];
          a.x += c.x;
          a.y += c.y;
          a.z += c.z;
          a.w += c.w;
        }
        s[0] = (a.x + a.y) + (a.z + a.w);
      } else {
#pragma unroll
        for (int k = 0; k < K; ++k) s[k] = buf[k][warp / kOfRow * kOfRow + lane % kOfRow];
#pragma unroll
        for (int m = kOfRow / 2; m >= 1; m >>= 1)
#pragma unroll
          for (int k = 0; k < K; ++k) s[k] += __shfl_xor_sync(0xffffffffu, s[k], m);
      }
    }
  }
  // the CTA's share of a sum over rows: out[col] of its line of the work buffer.  `stage`: kColumnBytes.
  __device__ __forceinline__ static void column_share(const F2 (&acc2)[P], float* out, float* stage, int t, int D) {
    float acc[N];
#pragma unroll
    for (int n = 0; n < P; ++n) {
      acc[2 * n] = lo(acc2[n]);
      acc[2 * n + 1] = hi(acc2[n]);
    }
    if constexpr (kRows == 1) {
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (col(t, n) < D) out[col(t, n)] = acc[n];
    } else {
      const int slot = threadIdx.x / T;
      __syncthreads();
#pragma unroll
      for (int n = 0; n < N; ++n) stage[slot * (T * N) + col(t, n)] = acc[n];
      __syncthreads();
      for (int c = threadIdx.x; c < D; c += kThreads) {
        float a = 0.f;
        for (int i = 0; i < kRows; ++i) a += stage[i * (T * N) + c];
        out[c] = a;
      }
    }
  }
};

// Rows ahead of the one in hand, in shared memory.  A thread copies and reads its own pieces only, so its own wait is all that stands
// between.  B: bytes of a thread and row; CTAS: CTAs on an SM, whose rings share what there is.
constexpr int ring_stages(int b, int threads_sm) {
  const int n = 196 * 1024 / (b * threads_sm);
  return n > 4 ? 4 : n;      // (three rows of 32 to 48 KB under way cover the latency)
}
template <typename S, int B, int CTAS, int SMALLEST> struct RowRing {      // SMALLEST: bytes of the smallest type of value
  static constexpr int kStages = S::W * SMALLEST >= 4 ? ring_stages(B, S::kThreads * CTAS) : 0;      // (2 bytes are no asynchronous copy)
  static constexpr bool kOn = kStages >= 2;      // else rows are loaded at the head of their turn
  static constexpr int kBytes = kOn ? kStages * B * S::kThreads : 0;
  unsigned char* base;
  __device__ __forceinline__ uint4* cell(int stage, int at) const { return reinterpret_cast<uint4*>(base) + (stage * (B / 16) + at) * S::kThreads + threadIdx.x; }
  // cells beyond the row are never copied to: zeros
  __device__ __forceinline__ explicit RowRing(unsigned char* smem) : base(smem) {
    if constexpr (kOn)
      for (int i = 0; i < kStages * (B / 16); ++i) *cell(0, i) = make_uint4(0, 0, 0, 0);
  }
  // this thread's pieces of a row to cells AT and on of a stage
  template <int TY, int AT>
  __device__ __forceinline__ void copy(int stage, const void* row, int t, int D) const {
    constexpr int kAll = S::W * elem_bytes(TY), kBytes = kAll > 16 ? 16 : kAll;
    const char* p = static_cast<const char*>(row);
#pragma unroll
    for (int m = 0; m < S::kMoves; ++m) {
      const int c = S::col(t, m * S::W);
      if (c >= D) continue;
#pragma unroll
      for (int k = 0; k < kAll; k += kBytes) {
        const int at = m * kAll + k;
        const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(cell(stage, AT + at / 16))) + at % 16;
        const char* from = p + static_cast<long long>(c) * elem_bytes(TY) + k;
        if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
        else if constexpr (kBytes >= 4) asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(kBytes) : "memory");
      }
    }
  }
  template <int TY, int AT>
  __device__ __forceinline__ void take(Raw<TY, 8> (&r)[S::R], int stage) const {
    constexpr int kEach = elem_bytes(TY) / 2;
#pragma unroll
    for (int i = 0; i < S::R; ++i)
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        const uint4 v = *cell(stage, AT + i * kEach + k);
        r[i].w[4 * k] = v.x;
        r[i].w[4 * k + 1] = v.y;
        r[i].w[4 * k + 2] = v.z;
        r[i].w[4 * k + 3] = v.w;
      }
  }
  // one group of copies for every row, also for those that are not there
  __device__ __forceinline__ static void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  __device__ __forceinline__ static void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kOn ? kStages - 2 : 0) : "memory"); }
};

// The turns of a thread: rows first, first + step, ...; all threads of a CTA take `all` of them, since row sums are collective, and
// have a row in the first `mine`.
struct Turns {
  long long first, step;
  int all, mine;
  __device__ __forceinline__ Turns(long long rows, int rows_per_cta, int slot) {
    const long long base = static_cast<long long>(blockIdx.x) * rows_per_cta;
    first = base + slot;
    step = static_cast<long long>(gridDim.x) * rows_per_cta;
    all = base < rows ? static_cast<int>((rows - base + step - 1) / step) : 0;
    mine = first < rows ? static_cast<int>((rows - first + step - 1) / step) : 0;
  }
};
// The place of a tensor's row, from turn to turn: additions only.
struct RowPtr {
  char* p;
  long long step;
  __device__ __forceinline__ RowPtr(const void* base, const Turns& t, long long stride, int bytes)
      : p(const_cast<char*>(static_cast<const char*>(base)) + t.first * stride * bytes), step(t.step * stride * bytes) {}
  __device__ __forceinline__ void next() { p += step; }
};
// Rows (o, i), i below `inner`, of tensors with a stride for each of the two.
struct RowWalk {
  uint32_t i, step_i, inner;      // (the sum of two numbers below inner < 2^31)
  long long o, step_o;
  __device__ __forceinline__ RowWalk(const Turns& t, long long inner_) : inner(static_cast<uint32_t>(inner_)) {
    o = t.first / inner_;
    i = static_cast<uint32_t>(t.first - o * inner_);
    step_o = t.step / inner_;
    step_i = static_cast<uint32_t>(t.step - step_o * inner_);
  }
  __device__ __forceinline__ bool next() {      // whether i has come round
    i += step_i;
    const bool round = i >= inner;
    if (round) i -= inner;
    return round;
  }
};
struct WalkPtr {
  char* p;
  long long step, round;
  __device__ __forceinline__ WalkPtr(const void* base, const RowWalk& w, long long outer, long long inner, int bytes)
      : p(const_cast<char*>(static_cast<const char*>(base)) + (w.o * outer + w.i * inner) * bytes), step((w.step_o * outer + w.step_i * inner) * bytes),
        round((outer - w.inner * inner) * bytes) {}
  __device__ __forceinline__ void next(bool come_round) { p += step + (come_round ? round : 0); }
};

// f(RowShape) for rows of D values: one piece of 8 a thread as far as a CTA goes.  With two, what a row costs beside its values (sums, places, loop)
// is shared by 16 of them, but half the threads are there to cover one another (us, one / two: gated 4 x 4096 x 16 x 128 bf16 forward
// 37.0 / 38.4, backward 66 / 71; residual 16384 x 4096 96 / 104; 64 rows of 2048 3.9 / 6.6).  Where 8 cannot be
// moved at once, fewer shapes.
template <int WIDEST, typename F>
int by_row_shape(int D, int w, F&& f) {
  const auto few = [&](auto n) {
    constexpr int W = decltype(n)::value;
    if (D <= 128) return f(RowShape<16, 1, W>());
    if (D <= 256) return f(RowShape<32, 1, W>());
    if (D <= 1024) return f(RowShape<128, 1, W>());
    if (D <= 4096) return f(RowShape<512, 1, W>());
    return f(RowShape<512, 2, W>());
  };
  if (w == 1) return few(std::integral_constant<int, 1>());
  if (w == 2) return few(std::integral_constant<int, 2>());
  if (w < WIDEST) return few(std::integral_constant<int, 4>());
  if (D <= 64) return f(RowShape<8, 1, WIDEST>());
  if (D <= 128) return f(RowShape<16, 1, WIDEST>());
  if (D <= 256) return f(RowShape<32, 1, WIDEST>());
  if (D <= 512) return f(RowShape<64, 1, WIDEST>());
  if (D <= 1024) return f(RowShape<128, 1, WIDEST>());
  if (D <= 2048) return f(RowShape<256, 1, WIDEST>());
  if (D <= 4096) return f(RowShape<512, 1, WIDEST>());
  return f(RowShape<512, 2, WIDEST>());
}
constexpr int widest_of(int t0, int t1) { return t0 == LETHE_F32 || t1 == LETHE_F32 ? 4 : 8; }

template <typename F>
int by_x_type(int xt, F&& f) {
  if (xt == LETHE_F32) return f(std::integral_constant<int, LETHE_F32>());
  if (xt == LETHE_BF16) return f(std::integral_constant<int, LETHE_BF16>());
  return f(std::integral_constant<int, LETHE_F16>());
}

inline bool norm_types_ok(int xt, int other) { return xt >= LETHE_F32 && xt <= LETHE_F16 && (other == LETHE_F32 || other == xt); }
// n values of type ty from ptr on can be moved at once, in every row
inline bool piece_aligned(int n, const void* ptr, int ty, long long s0 = 0, long long s1 = 0) {
  return reinterpret_cast<uintptr_t>(ptr) % (n * elem_bytes(ty)) == 0 && s0 % n == 0 && s1 % n == 0;
}
template <typename F>
int widest_piece(int widest, int D, F&& fits) {
  for (int n = widest; n > 1; n /= 2)
    if (D % n == 0 && fits(n)) return n;
  return 1;
}
inline int norm_grid(long long rows, int rows_per_cta, int ctas_per_sm) {
  const long long need = (rows + rows_per_cta - 1) / rows_per_cta;
  return static_cast<int>(std::min<long long>(need, static_cast<long long>(sm_count()) * ctas_per_sm));
}
inline int launched_ok() { return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch; }

// Sums the CTAs' shares: part[cta][vector][D] -> out[vector][D].
struct ColumnSums {
  const float* part;
  int parts, vectors, D;
  void* out[3];
  int f32[3], x_type;
};
int launch_column_sums(const ColumnSums& c, cudaStream_t st);

}  // namespace lg
