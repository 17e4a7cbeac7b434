// Element types of the operators that take their tensors as they are: fp32, bf16 or fp16 in memory, fp32 in registers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../../include/lethe_gdn.h"

namespace lg {

template <int TY> struct Elem;
template <> struct Elem<LETHE_F32> { using T = float; };
template <> struct Elem<LETHE_BF16> { using T = __nv_bfloat16; };
template <> struct Elem<LETHE_F16> { using T = __half; };

inline __host__ __device__ constexpr int elem_bytes(int ty) { return ty == LETHE_F32 ? 4 : 2; }
// whether all these pointers lie on a boundary of an element (null does)
template <typename... P> inline bool on_elements(int ty, const P*... p) { return ((reinterpret_cast<uintptr_t>(p) % elem_bytes(ty) == 0) && ...); }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
// one rounding, to nearest even
template <int TY> __device__ __forceinline__ typename Elem<TY>::T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<LETHE_F32>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<LETHE_BF16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f32<LETHE_F16>(float x) { return __float2half_rn(x); }

// Two floats that go through one instruction: each product and sum is rounded as by itself.
struct F2 { unsigned long long v; };
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ F2 f2(float a) { return f2(a, a); }
__device__ __forceinline__ float lo(F2 a) {
  float x, y;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v));
  return x;
}
__device__ __forceinline__ float hi(F2 a) {
  float x, y;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.v));
  return y;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// N neighbours as they lie in memory: read once, so they do not take room in L1.  The address is a multiple of their size (16 bytes at most).
template <int TY, int N> struct Raw {
  static constexpr int kWords = N * elem_bytes(TY) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void load(const typename Elem<TY>::T* p) {
    const uint32_t* s = reinterpret_cast<const uint32_t*>(p);
    if constexpr (kWords == 2) {
      asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(s));
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4)
        asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "l"(s + i));
    }
  }
  __device__ __forceinline__ void store(typename Elem<TY>::T* p) const {
    uint32_t* d = reinterpret_cast<uint32_t*>(p);
    if constexpr (kWords == 2) {
      *reinterpret_cast<uint2*>(d) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) *reinterpret_cast<uint4*>(d + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (TY == LETHE_F32) return __uint_as_float(w[i]);
    if constexpr (TY == LETHE_BF16) return __uint_as_float((i & 1) ? (w[i / 2] & 0xffff0000u) : (w[i / 2] << 16));
    if constexpr (TY == LETHE_F16) return __half2float(__ushort_as_half(static_cast<unsigned short>((i & 1) ? (w[i / 2] >> 16) : (w[i / 2] & 0xffffu))));
  }
  __device__ __forceinline__ F2 get2(int i) const { return f2(get(2 * i), get(2 * i + 1)); }      // pair i
  __device__ __forceinline__ void set2(int i, F2 a) { set2(2 * i, lo(a), hi(a)); }
  __device__ __forceinline__ void set2(int i, float a, float b) {      // elements i (even) and i + 1
    if constexpr (TY == LETHE_F32) {
      w[i] = __float_as_uint(a);
      w[i + 1] = __float_as_uint(b);
    }
    if constexpr (TY == LETHE_BF16) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
      w[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
    }
    if constexpr (TY == LETHE_F16) {
      const __half2 h = __floats2half2_rn(a, b);
      w[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
};

// 16-bit elements that are loaded one by one
template <int TY, int N>
__device__ __forceinline__ void raw_put(Raw<TY, N>& r, int i, typename Elem<TY>::T v) {
  if constexpr (TY == LETHE_F32) {
    r.w[i] = __float_as_uint(v);
  } else {
    const uint32_t b = *reinterpret_cast<const unsigned short*>(&v);
    r.w[i / 2] = (i & 1) ? ((r.w[i / 2] & 0xffffu) | (b << 16)) : ((r.w[i / 2] & 0xffff0000u) | b);
  }
}
template <int TY, int N>
__device__ __forceinline__ typename Elem<TY>::T raw_take(const Raw<TY, N>& r, int i) {
  if constexpr (TY == LETHE_F32) {
    return __uint_as_float(r.w[i]);
  } else {
    const unsigned short b = static_cast<unsigned short>((i & 1) ? (r.w[i / 2] >> 16) : (r.w[i / 2] & 0xffffu));
    return *reinterpret_cast<const typename Elem<TY>::T*>(&b);
  }
}

}  // namespace lg
