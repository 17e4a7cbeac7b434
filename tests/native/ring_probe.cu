// Self-test of the rings that move states (csrc/state_ring.cuh), and of their waits that give up.  Nothing faults and nothing hangs: a stage is armed for
// bytes that no copy brings, its wait ends after `limit_cycles`, the others' as soon as they see that, and the kernel returns.
#include "host_util.h"
#include "lethe_ring_probe.h"
#include "state_ring.cuh"

namespace lg {

constexpr int kProbeStrip = 512, kProbeStrips = 8;

__global__ void __launch_bounds__(256) ring_kernel(const char* in, char* out, int* status, int steps, int starved, int hole, long long limit, int* steps_of, int index) {
  __shared__ __align__(128) unsigned char memory[kCopyWarps * kStages * kProbeStrip];
  __shared__ RingMemory rings;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  Ring ring(rings, memory, kProbeStrip, status, 812);
  ring.ctl.limit = limit;
  if (index == 1 && threadIdx.x == 255) report(status, kErrIndex);
  __syncthreads();
  if (warp >= kCopyWarps) return;
  int i = 0;
  ring.run([&](int s, LaneCopy* c) {
    if (i >= steps) return false;
    const int strip = (warp * kProbeStrips + i % kProbeStrips) * kProbeStrip;
    ring.expect(s, kProbeStrip);
    const bool comes = i != hole || (starved != warp && starved != kCopyWarps);
    if (lane == 0 && comes) bulk_g2s(ring.stage(s), in + strip, kProbeStrip, ring.full + s);
    *c = LaneCopy{nullptr, 0, 0};
    if (lane == 0) *c = LaneCopy{out + strip, smem_u32(ring.stage(s)), kProbeStrip};
    ++i;
    return true;
  });
  steps_of[threadIdx.x] = i;
  if (index == 2) report(status, kErrIndex);
}

}  // namespace lg

extern "C" int lethe_probe_ring(const void* in, void* out, int* status, int steps, int starved, int hole, long long limit_cycles, int* steps_of, int index, void* stream) {
  using namespace lg;
  if (!in || !out || !status || !steps_of) return kErrNull;
  if (steps < 1 || steps > 200000 || starved < -1 || starved > kCopyWarps || limit_cycles < 1000 || limit_cycles > 200000000LL) return kErrDims;
  if ((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) % 16) return kErrAlign;
  ring_kernel<<<1, 256, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const char*>(in), static_cast<char*>(out), status, steps, starved, hole, limit_cycles, steps_of, index);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}
