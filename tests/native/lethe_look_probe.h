/* Test-only entry point of libletheprobe.so (tests/native/look_probe.cu): the bounded wait of the element-wise recurrence.  Not part of
 * the interface in include/lethe_gdn.h, no counterpart in the reference project. */
#ifndef LETHE_LOOK_PROBE_H_
#define LETHE_LOOK_PROBE_H_

#ifdef __cplusplus
extern "C" {
#endif

/* One CTA of 64 threads waits for 64 words that nobody writes, `words` of them all ones, with a limit of `limit_cycles` clock cycles (1e3 .. 2e8),
 * then waits for them again.  `head`: two 32-bit words, all ones.  Expected outcome: *status == 900, head[1] == 0 (everybody passes),
 * trace[0] ~ limit_cycles / 1024, trace[1] ~ 0 (the second wait fell through), got[0..63] == 0. */
int lethe_probe_look_wait(const void* words, void* head, int* status, long long limit_cycles, int* trace, unsigned long long* got, void* cuda_stream);

#ifdef __cplusplus
}
#endif
#endif
