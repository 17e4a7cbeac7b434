// Self-test of the bounded wait for a word (csrc/diag_look.cuh).  Nothing faults and nothing hangs: the words are memory of the caller that
// is never written, and the kernel ends by itself after `limit_cycles`.
#include "diag_look.cuh"
#include "host_util.h"
#include "lethe_look_probe.h"

namespace lg {

__global__ void __launch_bounds__(64) look_wait_kernel(const unsigned long long* words, uint32_t* head, int* status, long long limit, int* trace, unsigned long long* got) {
  const long long t0 = clock64();
  got[threadIdx.x] = look_wait(words + threadIdx.x, head, status, limit);
  __syncthreads();
  const long long t1 = clock64();
  got[threadIdx.x] |= look_wait(words + threadIdx.x, head, status, limit);
  __syncthreads();
  if (threadIdx.x == 0) {
    trace[0] = static_cast<int>((t1 - t0) / 1024);
    trace[1] = static_cast<int>((clock64() - t1) / 1024);
  }
}

}  // namespace lg

extern "C" int lethe_probe_look_wait(const void* words, void* head, int* status, long long limit_cycles, int* trace, unsigned long long* got, void* stream) {
  using namespace lg;
  if (!words || !head || !status || !trace || !got) return kErrNull;
  if (limit_cycles < 1000 || limit_cycles > 200000000LL) return kErrDims;      // at most a tenth of a second
  look_wait_kernel<<<1, 64, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const unsigned long long*>(words), static_cast<uint32_t*>(head), status, limit_cycles, trace, got);
  return cudaGetLastError() == cudaSuccess ? kOk : kErrLaunch;
}
