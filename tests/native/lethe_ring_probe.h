/* Test-only entry point of libletheprobe.so (tests/native/ring_probe.cu): the rings that move states.  Not part of the interface in
 * include/lethe_gdn.h, no counterpart in the reference project. */
#ifndef LETHE_RING_PROBE_H_
#define LETHE_RING_PROBE_H_

#ifdef __cplusplus
extern "C" {
#endif

/* One CTA whose four copying warps move strips of 512 bytes from `in` to `out` (4 x 8 strips each, step i of a warp its strip i % 8), up to `steps` of
 * them (1 to 200000).  `starved` (-1: none, 0 to 3: that warp, 4: all): arms its step `hole` for bytes that no copy brings, and waits for them with a limit of
 * `limit_cycles` clock cycles (1e3 .. 2e8).  steps_of[128]: the steps that each lane of these warps has begun.  Expected outcome of a starved warp: *status == 812,
 * a warp's lanes have the same number, those of the starved ones are hole + 4 at most, and the kernel has returned.
 * index (0: no): an index outside is reported too, 1: before the first step, 2: after the last. */
int lethe_probe_ring(const void* in, void* out, int* status, int steps, int starved, int hole, long long limit_cycles, int* steps_of, int index, void* cuda_stream);

#ifdef __cplusplus
}
#endif
#endif
