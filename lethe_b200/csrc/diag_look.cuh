// Words that tiles of the element-wise recurrence leave for one another (diag_scan.cu): 64 bits, stored and loaded as one, all ones where
// there is none yet.  Waiting for one is bounded.
#pragma once
#include <stdint.h>

namespace lg {

struct LookBuffer {
  uint32_t* head;                   // ticket, and the word that lets everybody pass
  unsigned long long* word[3];      // of tiles, groups of tiles, groups of groups
};
constexpr long long kLookLimitCycles = 2000000000LL;      // about one second
enum : int { kSiteLook = 900 };

__device__ __forceinline__ unsigned long long look_load(const unsigned long long* p) {
  unsigned long long v;
  asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void look_store(unsigned long long* p, float sum, float state) {
  unsigned long long v = (static_cast<unsigned long long>(__float_as_uint(state)) << 32) | __float_as_uint(sum);
  if (v == ~0ull) v = 0x7fffffff7fffffffull;      // (another NaN)
  asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}
__device__ __noinline__ unsigned long long look_wait(const unsigned long long* p, uint32_t* head, int* status, long long limit = kLookLimitCycles) {
  const long long t0 = clock64();
  for (int n = 1;; ++n) {
    const unsigned long long v = look_load(p);
    if (v != ~0ull) return v;
    if (n % 32) continue;
    if (*reinterpret_cast<volatile uint32_t*>(head + 1) == 0u) return 0;
    if (clock64() - t0 > limit) {
      atomicCAS(status, 0, kSiteLook);
      *reinterpret_cast<volatile uint32_t*>(head + 1) = 0u;
      return 0;
    }
  }
}

}  // namespace lg
