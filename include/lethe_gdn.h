/* C interface of liblethe_gdn.so: the chunked gated-delta-rule (GDN family) forward and backward on
 * NVIDIA B200 (sm_100a).
 *
 * It replaces, behind one pair of calls, what the reference project (RishiShah99/lethe) spreads over
 * its autograd op and its kernel plug-ins:
 *   - forward:  src/lethe/kernels/ops/gdn_layer.py:17-67 (_GDN2Function.forward, which today runs the
 *               token-serial src/lethe/kernels/references/gdn_backward.py:13-55 or the chunkwise
 *               restage src/lethe/kernels/references/gdn2_chunkwise_cw.py:213-314);
 *   - backward: src/lethe/kernels/ops/gdn_backward.py:16-57 -> src/lethe/kernels/cute/gdn2_backward.py:77-134
 *               -> src/lethe/kernels/cute/gdn2_assemble.py:242-314 / :601-696 / :711-775, i.e. the
 *               forward recompute, the reverse state scan K#1 (K1Fn, gdn2_assemble.py:29-32), the
 *               closed Stage B (:521-585) and the WY / triangular-inverse VJP K#2 (K2Fn, :33-44).
 *
 * Ownership: the caller allocates every buffer (inputs, outputs, the two workspaces and the status
 * word) on one GPU; the library works on the GPU that owns `q` (it need not be the calling thread's
 * current device), allocates nothing and keeps no state between calls.
 * Threading: re-entrant; all work is enqueued on the given stream; no call synchronises.
 * Errors: a non-zero return means nothing was launched (see lethe_gdn_strerror).  Device-side waits
 * are bounded; a wait that gave up leaves a non-zero code in *status, readable once the stream has
 * been synchronised (results are then invalid).  The caller zeroes *status before the first call.
 *
 * Layouts (all row-major, innermost dimension contiguous):
 *   q, k        [B, L, H, K]  bf16          v, o, do, dv [B, L, H, V]  bf16     dq, dk [B, L, H, K] bf16
 *               (q, k, dq, dk: fp16 when args->qk_f16 is set)
 *   g           [B, L, H] (gate = 1) or [B, L, H, K] (gate = 2), fp32, natural-log decay (<= 0)
 *   beta        [B, L, H] fp32 (delta = 1)
 *   h0, hT, dhT, dh0   [B, H, K, V] fp32
 *   dg          like g, fp32;   dbeta like beta, fp32
 * Sizes: dims.K = 128, dims.V in {64, 128}, dims.L a multiple of 64 (the chunk length); tensors with 64 key
 * channels or another number of tokens say so in k_channels and l_tokens.
 */
#ifndef LETHE_GDN_H_
#define LETHE_GDN_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { LETHE_GATE_NONE = 0, LETHE_GATE_SCALAR = 1, LETHE_GATE_CHANNEL = 2 };

typedef struct LetheGdnDims {
  int32_t B, H, L, K, V;
  int32_t gate;   /* LETHE_GATE_*                                                        */
  int32_t delta;  /* 1: erase and write gates are beta (gated delta rule, KDA)            */
                  /* 0: no erase term, write gate one (linear attention, GLA, SSD)        */
                  /* 2: independent per-channel erase gate b and write gate w, the full   */
                  /*    op of the reference (gdn_backward.py:45-53); needs the            */
                  /*    channel-wise gate                                                 */
} LetheGdnDims;

typedef struct LetheGdnArgs {
  LetheGdnDims dims;
  float scale;            /* multiplies q; the reference default is K^-0.5                  */
  /* forward inputs */
  const void* q;
  const void* k;
  const void* v;
  const float* g;         /* NULL when gate == LETHE_GATE_NONE                              */
  const float* beta;      /* NULL when delta == 0                                           */
  const float* h0;        /* NULL: zero initial state                                       */
  /* forward outputs */
  void* o;
  float* hT;              /* NULL: final state not wanted                                   */
  /* backward inputs */
  const void* d_o;
  const float* dhT;       /* NULL: zero                                                     */
  /* backward outputs */
  void* dq;
  void* dk;
  void* dv;
  float* dg;              /* NULL when gate == LETHE_GATE_NONE                              */
  float* dbeta;           /* NULL when delta == 0                                           */
  float* dh0;             /* NULL: not wanted                                               */
  /* caller-owned scratch */
  void* saved;            /* written by forward, read by backward; lethe_gdn_saved_bytes     */
  size_t saved_bytes;
  void* scratch;          /* backward only; lethe_gdn_scratch_bytes                          */
  size_t scratch_bytes;
  int32_t* status;        /* device word, see above                                         */
  /* Profiling aid: 0 runs every kernel of the call.  Otherwise bit i selects kernel i of the call  */
  /* (forward: 1 prepare, 2 state scan, 4 output; backward: 1 scan input, 2 adjoint scan,           */
  /* 4 Stage B, 8 WY VJP); a partial call relies on the records left by an earlier full call (names   */
  /* and layout: csrc/gdn_common.cuh) - one with lean 0, where a scan of the full call would be joint  */
  /* with the kernel beside it (lethe_gdn_joint_scans): a lean full call then leaves no RB behind the  */
  /* adjoint and, with lean 2, no Hc behind the forward.  A partial call that has one of the two       */
  /* kernels but not the other runs it by itself, lean or not.                                        */
  /* Backward with the delta term, records read: 1: A (of TA), W,                                      */
  /* QG (channel-wise gate); 2: P, AD, RB; 4: A, VN, Hc, DH; 8: T (of TA), W and U (the WY factors     */
  /* w = T (beta gamma k) and u = T (beta v), which the gradient of the inverse is formed with), and   */
  /* DV2, DW, DKB, DGB, RB as bit 4 left them.  A caller that lays records down for 8 alone has to     */
  /* supply W and U too.  Without the delta term 4 reads A, Hc and DH, and 8 is empty.                 */
  uint32_t kernel_mask;
  /* Optional split of the beta gradient (delta = 1).  NULL: `dbeta` receives the whole gradient.     */
  /* Non-NULL: `dbeta` receives the erase-gate part and `dbeta_write` the write-gate part, the two    */
  /* gradients the reference returns separately (db_erase / dw_write, gdn2_assemble.py:150-181).      */
  float* dbeta_write;
  /* delta = 2 only (NULL otherwise): erase gate b [B, L, H, K] and write gate w [B, L, H, V], fp32,     */
  /* and their gradients (backward).  `beta` / `dbeta` are not used in this mode.                       */
  const float* b_gate;
  const float* w_gate;
  float* db_gate;
  float* dw_gate;
  /* The (batch, head) pairs this call works on: pairs [bh_begin, bh_begin + bh_count) in b * H + h order;     */
  /* bh_count = 0 means all of them.  Pairs are independent recurrences: calls on disjoint ranges may run     */
  /* concurrently on different streams with the same tensors and workspaces (no counterpart in the reference). */
  uint32_t bh_begin;
  uint32_t bh_count;
  /* Non-zero: q, k (inputs) and dq, dk (outputs) hold IEEE fp16 instead of bf16.  fp16 is the type of the  */
  /* tensor-core operands, so a caller that forms q, k in fp32 (the L2 normalisation below) rounds them      */
  /* once, as the reference does when it stages operands (gdn2_bwd_dhu_l3.py:477-479), instead of twice.     */
  /* v, o, d_o, dv stay bf16.                                                                               */
  uint32_t qk_f16;
  /* The chunks (64-token blocks) of every sequence this call works on: [c_begin, c_begin + c_count); c_count = 0  */
  /* means all L / 64 of them.  The chunk-parallel kernels simply cover that range.  The state scans carry    */
  /* their fp32 state from one range to the next through the workspaces, so the forward ranges must be run    */
  /* in ascending order and the backward ranges in descending order (kernel_mask selects the kernels): a      */
  /* call cut into ranges gives bit-identical results and lets a caller overlap the chunk-parallel kernels    */
  /* of one range with the serial scan of the next on another stream (lethe_b200.ops.GdnStepGraph does).      */
  /* No counterpart in the reference.                                                                          */
  uint32_t c_begin;
  uint32_t c_count;
  /* Sequences that do not fill their last chunk, and 64 key channels (delta 0 or 1).  dims.L stays a multiple of  */
  /* 64 and dims.K 128 (they size the workspaces); l_tokens in (dims.L - 64, dims.L] and k_channels = 64 say how   */
  /* many tokens and key channels the tensors really have, in the same layouts ([B, l_tokens, H, k_channels] ...,  */
  /* states [B, H, k_channels, V]).  The rest counts as zero and is neither read nor written.  0: all of dims.     */
  uint32_t l_tokens;
  uint32_t k_channels;
  /* 1: the call leaves only results in memory, and in the workspaces what its own later kernels and, after a forward, */
  /* the backward read.  2 (forward only): not even the latter, no backward can follow.  0: also intermediates that a  */
  /* caller may want to look at (dv2, dw), and whatever a partial call (kernel_mask) on the same workspaces may read:  */
  /* a lean call may do the work of two kernels in one, and what goes between them is then not written.                */
  uint32_t lean;
  /* Forward.  l2_eps > 0: q and k are normalised as they are read, x rsqrt(sum x^2 + l2_eps) per token-head, in fp32   */
  /* and rounded once to fp16 (what lethe_gdn_l2norm_qk does, without its pass over memory).  q_norm, k_norm take the     */
  /* normalised rows, fp16, for the backward: both or neither with LETHE_GATE_CHANNEL; otherwise q_norm is needed (the   */
  /* output kernel reads it) and k_norm is for a backward.                                                                */
  float l2_eps;
  void* q_norm;
  void* k_norm;
} LetheGdnArgs;

/* Bytes of the forward->backward workspace / of the backward scratch for these sizes (0 = bad dims). */
size_t lethe_gdn_saved_bytes(const LetheGdnDims* dims);
size_t lethe_gdn_scratch_bytes(const LetheGdnDims* dims);

/* Which scans of whole calls on these sizes do the work of the kernel beside them (output kernel, scan input) themselves, on a    */
/* GPU of `sms` SMs (0: the current device): one launch less each, and the records between the two are not written.  0 for lean 0.  */
/* No counterpart in the reference.                                                                                                */
enum { LETHE_JOINT_FORWARD = 1, LETHE_JOINT_ADJOINT = 2 };
int lethe_gdn_joint_scans(const LetheGdnDims* dims, uint32_t lean, int32_t sms);

/* Forward: o (and hT) from q, k, v, g, beta, h0.  Replaces gdn_layer.py:17-67 of the reference. */
int lethe_gdn_forward(const LetheGdnArgs* args, void* cuda_stream);

/* Backward: dq, dk, dv, dg, dbeta, dh0 from the forward inputs, d_o, dhT and `saved`.
 * Replaces gdn_backward.py:16-57 / gdn2_assemble.py:242-314,601-696,711-775 of the reference. */
int lethe_gdn_backward(const LetheGdnArgs* args, void* cuda_stream);

/* Forward without a caller-supplied workspace, for hosts that cannot allocate device memory (a
 * plug-in inside a runtime whose memory pool is off limits, a server that fixed its memory budget
 * at start-up).  It has no counterpart in the reference.  Same arguments and results as
 * lethe_gdn_forward, except that args->saved / saved_bytes are ignored: the per-chunk records go
 * through a 16 MiB array built into the library (lethe_gdn_forward_static_capacity()), so
 *   - the problem must satisfy lethe_gdn_saved_bytes(dims) <= 16 MiB, else the call returns the
 *     "needs more workspace" error and launches nothing;
 *   - the records are not kept for a backward pass (inference / evaluation only);
 *   - all calls on one GPU share the array: calls that could overlap on the GPU must be put on one
 *     stream; nothing needs clearing between calls;
 *   - every GPU has its own copy of the array.  The call works on the GPU that owns args->q,
 *     whatever device the calling thread has selected, and uses that GPU's copy;
 *   - the first call for each GPU looks up the array's device address there and may make the driver
 *     load the library's code onto that GPU (this is when the 16 MiB get reserved); make that call
 *     before any stream capture starts.
 * After that first call on a GPU, a call allocates nothing (no cudaMalloc, no cudaFree, no library
 * that would). */
int lethe_gdn_forward_static(const LetheGdnArgs* args, void* cuda_stream);
size_t lethe_gdn_forward_static_capacity(void);

/* One token of the same recurrence for generation (the body of the reference's token loop,
 * src/lethe/kernels/references/gdn_backward.py:45-53; the reference has no device kernel for it):
 *   S <- S * exp(g);  v_new = beta (v - k^T S);  S <- S + k v_new^T;  o = (scale q)^T S
 * for every (batch, head) pair.  q, k: bf16 [B, H, K]; v, o: bf16 [B, H, V]; g: fp32 [B, H] (scalar
 * gate) or [B, H, K] (channel-wise), unused for LETHE_GATE_NONE; beta: fp32 [B, H], required when
 * delta != 0; state: fp32 [B, H, K, V], updated in place (the h_T of lethe_gdn_forward continues a
 * prompt).  K = 128, V in {64, 128}.  No workspace, no status word (the kernel waits on nothing). */
typedef struct LetheGdnDecodeArgs {
  int32_t B, H, K, V;
  int32_t gate;   /* LETHE_GATE_* */
  int32_t delta;  /* 0: no delta term (v_new = v) */
  float scale;
  const void* q;
  const void* k;
  const void* v;
  const float* g;
  const float* beta;
  float* state;
  void* o;
  uint32_t in_f32;   /* non-zero: q, k, v are fp32; each value is rounded to bf16 as it is read */
} LetheGdnDecodeArgs;
int lethe_gdn_decode_step(const LetheGdnDecodeArgs* args, void* cuda_stream);

/* L2 normalisation of q and k before the recurrence, and its vector-Jacobian product after the
 * backward (reference src/lethe/kernels/references/gdn_backward.py:9-10, applied at :29-31 when
 * use_qk_l2norm is set; the reference differentiates it by autograd,
 * src/lethe/kernels/references/gdn2_assemble.py:300-312):
 *   y = x * rsqrt(sum_d x_d^2 + eps);      dx = r (dy - y (y . dy)),  r = rsqrt(sum_d x_d^2 + eps).
 * flags: LETHE_L2_IN_F32  - q, k (and the returned dq, dk) are fp32 instead of bf16;
 *        LETHE_L2_IN_F16  - ... fp16 (at most one of the two);
 *        LETHE_L2_NORM_F16 - the normalised rows qn, kn and their gradients dqn, dkn are fp16 instead
 *                            of bf16 (pair it with LetheGdnArgs::qk_f16 on the forward / backward
 *                            calls: the rows are then rounded once, to the operand type);
 *        LETHE_L2_EARLY   - VJP only: the call directly follows lethe_gdn_backward on its stream and q, k are older
 *                            than that call; they are read before its last kernel has ended.
 * q, k: [rows, D] contiguous; D in {64, 128}; rows = B L H.
 * qn, kn: 16-bit [rows, D], the tensors lethe_gdn_forward / lethe_gdn_backward then read.
 * dqn, dkn: 16-bit [rows, D], the dq / dk lethe_gdn_backward wrote; dq, dk: [rows, D] in the type of
 * q, k (may alias dqn, dkn when both are bf16).  One launch each; every pointer 16-byte aligned. */
enum { LETHE_L2_IN_F32 = 1, LETHE_L2_NORM_F16 = 2, LETHE_L2_IN_F16 = 4, LETHE_L2_EARLY = 8 };
int lethe_gdn_l2norm_qk(const void* q, const void* k, void* qn, void* kn, int64_t rows, int32_t D,
                        int32_t flags, float eps, void* cuda_stream);
int lethe_gdn_l2norm_qk_vjp(const void* q, const void* k, const void* dqn, const void* dkn, void* dq, void* dk,
                            int64_t rows, int32_t D, int32_t flags, float eps, void* cuda_stream);

/* The six-input surface of the reference (gdn_layer.py:99-111) takes every gate per channel: g, b [rows, K], w
 * [rows, V], fp32, rows = B L H.  lethe_gdn_gate_regime decides which kernels such a call needs, as the reference
 * does (cute/gdn2_backward.py:53-60), by bitwise comparison along the channels, and compacts what those kernels read:
 *   *flags (4-byte device or mapped host word) = LETHE_REGIME_DONE | the tests that hold:
 *     SCALAR_GATE  g is one value per row;   ONE_BETA  b and w are the same one value per row;
 *     NO_DELTA     b is 0 and w is 1 everywhere;
 *   g0 [rows], b0 [rows]: g[:, 0] and b[:, 0], complete when one of the tests that use them holds.
 * work: 8 bytes of device memory, zero before the call and again after it.
 * lethe_gdn_gate_spread is the other direction: gradients per row spread evenly over the channels, as the reference's
 * scalar assembly does (gdn2_assemble.py:343-345): dg[r, :] = dg0[r] / K, db[r, :] = db0[r] / K, dw[r, :] = dw0[r] / V.
 * A null output is not wanted, a null source counts as zero. */
enum { LETHE_REGIME_SCALAR_GATE = 1, LETHE_REGIME_ONE_BETA = 2, LETHE_REGIME_NO_DELTA = 4, LETHE_REGIME_DONE = 8 };
int lethe_gdn_gate_regime(const float* g, const float* b, const float* w, int64_t rows, int32_t K, int32_t V,
                          float* g0, float* b0, uint32_t* flags, uint32_t* work, void* cuda_stream);
int lethe_gdn_gate_spread(const float* dg0, const float* db0, const float* dw0, int64_t rows, int32_t K, int32_t V,
                          float* dg, float* db, float* dw, void* cuda_stream);

/* n values from bf16 to fp32 (to_f32 != 0) or from fp32 to bf16, rounded to nearest even; both pointers on 16-byte     */
/* boundaries.  No counterpart in the reference.                                                                        */
int lethe_gdn_convert(const void* src, void* dst, int64_t n, int32_t to_f32, void* cuda_stream);

/* ------------------------------------------------------------------------------------------------------------------
 * What stands beside a recurrence with a matrix state in a model: the recurrence with one state value per channel, and the
 * norms on both sides of a block.  No counterpart in the reference.  These calls take tensors in the type they have
 * (LETHE_F32, LETHE_BF16, LETHE_F16), compute in fp32 and round each result once.  Strides and offsets count elements;
 * rows are read where they lie, the innermost dimension contiguous; pointers on a boundary of their element (else refused).  Like the
 * calls above they allocate nothing, enqueue on the given stream and return non-zero where nothing was launched; they work
 * on the GPU that owns `x`.
 * ------------------------------------------------------------------------------------------------------------------ */
enum { LETHE_F32 = 0, LETHE_BF16 = 1, LETHE_F16 = 2 };

/* The element-wise gated recurrence, for every sequence b and channel d:
 *   h_t = exp(g_t) h_{t-1} + x_t                       (complement != 0: exp(g_t) h_{t-1} + (1 - exp(g_t)) x_t)
 * forward: h and hT from x, g, h0.  backward, with e_t the gradient of h_t: e_t = d_h_t + exp(g_{t+1}) e_{t+1},
 *   dx_t = e_t (times 1 - exp(g_t)),  dg_t = exp(g_t) e_t (h_{t-1} (- x_t)),  dh0 = exp(g_0) e_0.
 * g is a natural-log decay, <= 0; minus infinity starts anew.  What is not finite reaches all later tokens of its channel, also
 * past such a start, and an infinite state may go on as NaN.  States are fp32; the decay of a long memory keeps its
 * precision (1 - exp(g) is formed without the cancellation that exp(g) next to one would bring).
 * Types: x, h, d_h, dx are x_type; g, dg are g_type, which is LETHE_F32 or x_type.  h0, hT, dhT, dh0 fp32 [B, D].
 * h, dx, dg are contiguous [B, L, D]; x, g, d_h have strides of their own for batch and token.
 * states: fp32, lethe_gdn_diag_states_bytes; the forward writes it where it is not NULL, the backward reads it.
 * work: lethe_gdn_diag_work_bytes bytes on a 16-byte boundary, scratch of one call (NULL where that is 0).
 * status: as above; a device-side wait that gave up leaves a non-zero code there. */
typedef struct LetheGdnDiagArgs {
  int64_t B, L, D;
  int32_t x_type, g_type, complement;
  const void* x;
  int64_t x_batch, x_token;
  const void* g;
  int64_t g_batch, g_token;
  const float* h0;        /* NULL: zero                                                     */
  void* h;                /* forward                                                        */
  float* hT;              /* NULL: not wanted                                               */
  float* states;          /* forward: NULL where no backward follows                        */
  const void* d_h;        /* backward; NULL: zero                                           */
  int64_t d_h_batch, d_h_token;
  const float* dhT;       /* NULL: zero                                                     */
  void* dx;               /* NULL: not wanted, as dg and dh0                                */
  void* dg;
  float* dh0;
  void* work;
  size_t work_bytes;
  int32_t* status;
} LetheGdnDiagArgs;
size_t lethe_gdn_diag_states_bytes(int64_t B, int64_t L, int64_t D, int32_t x_type);
size_t lethe_gdn_diag_work_bytes(int64_t B, int64_t L, int64_t D, int32_t x_type, int32_t backward);
int lethe_gdn_diag_forward(const LetheGdnDiagArgs* args, void* cuda_stream);
int lethe_gdn_diag_backward(const LetheGdnDiagArgs* args, void* cuda_stream);

/* One token of it for generation: state [B, D] fp32, contiguous, updated in place; h [B, D] contiguous in x_type.  Uses B, D,
 * the types, x, g and their batch strides. */
int lethe_gdn_diag_step(const LetheGdnDiagArgs* args, float* state, void* cuda_stream);

/* The norm behind a block: y = x rsqrt(mean(x^2) + eps) weight act(gate), act the logistic function, or gate times it (silu != 0).
 * Norm first, gate behind.  Rows of D values, 1 <= D <= 8192: row r = i * inner + j (inner below 2^31) lies at i * outer_stride + j * inner_stride, for x and gate each;
 * y, dx, dgate are contiguous.  x, gate, y, dy, dx, dgate are x_type; weight and dweight LETHE_F32 or x_type (w_type).
 * dy contiguous.  work (vjp): lethe_gdn_norm_work_bytes(rows, D, 1) bytes on a 16-byte boundary, needed where dweight is wanted. */
typedef struct LetheGdnGatedNormArgs {
  int64_t rows, inner;
  int32_t D, x_type, w_type, silu;
  float eps;              /* finite, zero or more                                           */
  const void* x;
  int64_t x_outer, x_inner;
  const void* gate;
  int64_t gate_outer, gate_inner;
  const void* weight;
  void* y;
  const void* dy;
  void* dx;               /* NULL: not wanted, as dgate and dweight                         */
  void* dgate;
  void* dweight;
  void* work;
  size_t work_bytes;
} LetheGdnGatedNormArgs;
int lethe_gdn_gated_norm(const LetheGdnGatedNormArgs* args, void* cuda_stream);
int lethe_gdn_gated_norm_vjp(const LetheGdnGatedNormArgs* args, void* cuda_stream);

/* The residual sum and the norm in front of the next block:
 *   t = x  or, with post_weight,  x rsqrt(mean(x^2) + eps) post_weight;     r = residual + scale t, rounded to r_type;
 *   y = r rsqrt(mean(r^2) + eps) weight       (of r as it was rounded, so that every later reader of r sees the same).
 * scale: a vector of D values, or NULL for the number scale_value.  residual NULL: zero.
 * x, y, dy, dx are x_type; residual, r, dr, dresidual r_type (LETHE_F32 or x_type); weight, post_weight, scale and their
 * gradients w_type (LETHE_F32 or x_type).  Rows of D values, 1 <= D <= 8192; x and residual have a stride between rows, the rest is contiguous.
 * vjp: reads r as the forward wrote it, x where post_weight or dscale needs it, dy and dr (either may be NULL: zero).
 * work (vjp): lethe_gdn_norm_work_bytes(rows, D, n) bytes on a 16-byte boundary, n the number of vector gradients wanted. */
typedef struct LetheGdnResidualNormArgs {
  int64_t rows;
  int32_t D, x_type, r_type, w_type;
  float eps, scale_value;   /* eps: finite, zero or more                                      */
  const void* x;
  int64_t x_stride;
  const void* residual;
  int64_t residual_stride;
  const void* weight;
  const void* post_weight;  /* NULL: no norm of x                                           */
  const void* scale;
  void* r;
  void* y;
  const void* dy;
  const void* dr;
  void* dx;                 /* NULL: not wanted, as the other gradients                     */
  void* dresidual;
  void* dweight;
  void* dpost_weight;
  void* dscale;
  void* work;
  size_t work_bytes;
} LetheGdnResidualNormArgs;
size_t lethe_gdn_norm_work_bytes(int64_t rows, int32_t D, int32_t vectors);
int lethe_gdn_residual_norm(const LetheGdnResidualNormArgs* args, void* cuda_stream);
int lethe_gdn_residual_norm_vjp(const LetheGdnResidualNormArgs* args, void* cuda_stream);

/* ------------------------------------------------------------------------------------------------------------------
 * Decoding with several hypotheses: choosing tokens, and moving the states that belong to them.  No counterpart in the reference.
 * These calls work on the GPU that owns `logits`, the first tensor of states (fork and compact: `live`), or `state`, and otherwise as the ones above.
 * ------------------------------------------------------------------------------------------------------------------ */

/* Beam search's selection: for B groups of W beams over V tokens,
 *   c_wv = scores_w + l_wv / temperature - log sum_u exp(l_wu / temperature)   over the allowed tokens,
 * the k candidates (w, v) with the largest c_wv / penalty_w, in order, of equal ones the lowest (w, v) first.  A finished beam offers
 * itself, with its score, at the token eos and nothing else.  A beam offers nothing whose score is not finite, whose penalty is not
 * above zero and finite, or that has no distribution (no allowed token above minus infinity, NaN or plus infinity at an allowed one).
 * Candidates are ordered as in 64 bits.  Where there are fewer than k the rest has score minus infinity, parent 0, token eos
 * (0 without eos) and counts as finished.
 * logits [B, W, V] x_type, allowed bytes (non-zero: allowed), both with strides for group and beam (0: shared) in elements;
 * scores, penalty fp32 [B, W], finished bytes [B, W], out_* [B, k].  W, k from 1 to 64, V to 2^30, temperature 1e-6 to 1e6.
 * work: lethe_gdn_beam_work_bytes bytes on a 16-byte boundary, scratch of one call.
 * Results and work lie apart from one another and from the inputs (refused otherwise for all but logits and allowed); with k = W out_scores may be scores
 * or penalty, and out_finished may be finished. */
typedef struct LetheGdnBeamArgs {
  int64_t B, V;
  int32_t W, k, x_type;
  double temperature;
  const void* logits;
  int64_t logits_batch, logits_beam;
  const uint8_t* allowed;   /* NULL: every token                                              */
  int64_t allowed_batch, allowed_beam;
  const float* scores;
  const uint8_t* finished;  /* NULL: none                                                     */
  const float* penalty;     /* NULL: one                                                      */
  int64_t eos;              /* -1: none (neither finished nor out_finished then)              */
  float* out_scores;        /* c, not divided by the penalty                                  */
  int64_t* parents;
  int64_t* tokens;
  uint8_t* out_finished;    /* NULL: not wanted.  Whether the parent was, or the token is eos  */
  void* work;
  size_t work_bytes;
} LetheGdnBeamArgs;
size_t lethe_gdn_beam_work_bytes(int64_t B, int32_t W, int64_t V, int32_t k, int32_t x_type);
int lethe_gdn_beam_select(const LetheGdnBeamArgs* args, void* cuda_stream);

/* States of sequences: for each of `count` tensors a row of row_bytes bytes per sequence, of any type, at
 * data + group * group_stride + i * stride (bytes; whole rows do not overlap), row_bytes up to 2^38.  `states` is host memory, read during the call. */
typedef struct LetheGdnStates {
  void* data;
  int64_t row_bytes, stride, group_stride;
} LetheGdnStates;

/* Row (b, w) becomes what row (b, parents[b, w]) was, in every tensor at once and in place, for B groups of W rows (W to 256).
 * parents [B, W], int64 or (parents_64 = 0) int32.  A parent outside [0, W) leaves its row as it was and a code in *status. */
int lethe_gdn_reorder_states(const LetheGdnStates* states, int32_t count, int64_t B, int32_t W, const void* parents, int32_t parents_64,
                             int32_t* status, void* cuda_stream);

/* A pool of slots (rows i of every tensor, to 65536; group_stride unused), live[i] non-zero for the ones in use.
 * fork: n entries (to 4096); entry e takes the lowest free slot that no entry in front of it takes, target[e], which gets the values of
 *   slot source[e] (zeros where that is -1).  Where source[e] is neither -1 nor a live slot, or no slot is left, target[e] = -1 and
 *   nothing is taken.  live_after = live and the slots taken.  source int64 or (source_64 = 0) int32.
 * compact: the m live slots become slots 0 to m - 1: the ones at or behind m, in their order, move to the free ones in front of m, in
 *   theirs; what lies behind is left as it was.  place[i] = the new slot of live slot i, -1 for others; *live_count = m.
 * Results lie apart from live and source and from one another (refused otherwise), and all of these apart from the states' rows. */
int lethe_gdn_fork_states(const LetheGdnStates* states, int32_t count, int64_t slots, const uint8_t* live, const void* source, int32_t source_64,
                          int64_t n, int64_t* target, uint8_t* live_after, int32_t* status, void* cuda_stream);
int lethe_gdn_compact_states(const LetheGdnStates* states, int32_t count, int64_t slots, const uint8_t* live, int64_t* place,
                             int64_t* live_count, int32_t* status, void* cuda_stream);

/* lethe_gdn_decode_step with a state of its own for what it writes: row b goes on from row source[b] of args->state [slots, H, K, V]
 * (-1: from zeros), and its new state is row b of out [B, H, K, V], memory apart from everything else of the call (refused otherwise).  source [B], int64 or
 * (source_64 = 0) int32; one outside [-1, slots) gives NaN and a code in *status. */
int lethe_gdn_decode_step_from(const LetheGdnDecodeArgs* args, int64_t slots, const void* source, int32_t source_64, float* out,
                               int32_t* status, void* cuda_stream);

/* Text for a return code of the calls above or for a device status code. */
const char* lethe_gdn_strerror(int code);

#ifdef __cplusplus
}
#endif
#endif /* LETHE_GDN_H_ */
