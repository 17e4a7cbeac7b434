// Rings of strips in shared memory, global memory to global memory by bulk copies: a warp that issues them has a ring of its own, and no thread touches
// the data.
#pragma once
#include "host_util.h"
#include "umma.cuh"

namespace lg {

constexpr int kCopyWarps = 4;
// Stages of a ring: as many strips on their way in as out.  A compaction of 543 MB (83 us at the copy rate) in us:
// four rings of 8 KB strips 93, two of 16 KB 92, four of 2 KB 134, one of 16 KB with two strips on their way out 101, without rings, through registers, 98.
constexpr int kStages = 6, kOut = kStages / 2;

// A warp's ring.  Lane 0 expects what comes; a stage is filled again when the stores out of it have read it.
struct LaneCopy {           // what a lane stores out of a stage
  char* to;
  uint32_t from, bytes;     // (0: nothing)
};
struct RingMemory {
  uint64_t full[kCopyWarps][kStages];
  LaneCopy copies[kCopyWarps][kStages][32];
  int abort_flag;
};

struct Ring {
  unsigned char* bytes;
  uint64_t* full;
  LaneCopy (*copies)[32];
  CtaCtl ctl;
  int stage_bytes, site;
  uint32_t phases = 0, filled = 0;      // bit s: the parity that stage s is waited for next; loads into it that nobody has waited for

  // (all threads of the CTA, in front of a barrier)
  __device__ __forceinline__ Ring(RingMemory& m, unsigned char* memory, int stage_bytes, int* status, int site)
      : bytes(memory + threadIdx.x / 32 % kCopyWarps * kStages * stage_bytes), full(m.full[threadIdx.x / 32 % kCopyWarps]),
        copies(m.copies[threadIdx.x / 32 % kCopyWarps]), ctl{status, &m.abort_flag}, stage_bytes(stage_bytes), site(site) {
    if (threadIdx.x < kCopyWarps * kStages) mbar_init(&m.full[0][0] + threadIdx.x, 1);
    if (threadIdx.x == 0) m.abort_flag = 0;
    fence_mbar_init();
  }
  __device__ __forceinline__ unsigned char* stage(int s) const { return bytes + s * stage_bytes; }
  __device__ __forceinline__ void expect(int s, uint32_t n) {
    if (threadIdx.x % 32 == 0) mbar_expect_tx(full + s, n);
    filled |= 1u << s;
    __syncwarp();
  }
  // Whether the loads of a stage are there.  Where a wait of the CTA gave up they may not be: the warp then waits, with a limit, for whatever is still on
  // its way into the ring, that stage's among it, before it leaves.  One lane may see the flag of another warp before the next does, so
  // the warp decides as one.
  __device__ __forceinline__ bool arrive(int s) {
    const uint32_t bit = filled & (1u << s);
    if (bit) mbar_wait_warp(full + s, (phases >> s) & 1, ctl, site);
    if (__any_sync(~0u, *ctl.abort_flag)) {
      atomicCAS(ctl.status, kErrIndex, site);      // (an index outside spoils its own rows only: the wait is what the host has to hear of)
      const long long t0 = clock64();
      for (int i = 0; i < kStages; ++i)
        while (((filled >> i) & 1) && !mbar_try(full + i, (phases >> i) & 1) && clock64() - t0 < ctl.limit) {
        }
      __syncwarp();
      return false;
    }
    phases ^= bit;
    filled ^= bit;
    return true;
  }

  // Step after step: load(s, &copy) issues the next one's copies into stage s and says what the lane stores out of it, or that there is none.
  template <typename Load> __device__ __forceinline__ void run(Load load) {
    const int lane = threadIdx.x % 32;
    int loaded = 0, into = 0, at = 0;
    bool more = true;
    auto one = [&] {
      LaneCopy c;
      more = load(into, &c);
      if (!more) return;
      copies[into][lane] = c;
      into = into + 1 == kStages ? 0 : into + 1;
      ++loaded;
    };
    while (more && loaded < kStages - kOut) one();
    for (int stored = 0; stored < loaded; ++stored) {
      if (more) {      // (the stage that `kOut` steps ago was stored from)
        asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kOut - 1) : "memory");
        __syncwarp();
        one();
      }
      if (!arrive(at)) break;
      const LaneCopy c = copies[at][lane];
      if (c.bytes) asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(c.to), "r"(c.from), "r"(c.bytes) : "memory");
      bulk_commit();
      at = at + 1 == kStages ? 0 : at + 1;
    }
    bulk_wait_read();
  }
};

}  // namespace lg
