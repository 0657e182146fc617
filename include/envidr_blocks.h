/*
 * envidr_amd -- C-ABI of the block operators: what a learnt block over packed ray samples needs beside the dense layers and the
 * compositors of envidr_amd.h / envidr_render.h.  No reference counterpart.
 *
 *   envidr_gated_mlp_*       y = (act(x Wg^T) * (x Wu^T)) Wd^T and its gradients
 *   envidr_ray_recurrence_*  h_t = a_t h_{t-1} + s_t v_t along every ray's samples, a_t = sigmoid(gate_t), and its gradients
 *   envidr_dropout*          counter-based dropout (the mask is recomputed, never stored), with a residual sum
 *
 * Conventions: those of envidr_amd.h (device pointers, asynchronous on `stream`, 0 or a negative ENVIDR_E* code and
 * envidr_last_error(), an empty batch is a successful no-op), and
 *   - `dtype` is one of ENVIDR_F32 / ENVIDR_BF16 / ENVIDR_F16 and holds for every `void*` tensor of a call; sums, activations and
 *     states are computed in 32 bits or more and rounded once where they are stored;
 *   - a row pitch (`ld*`) counts elements, the elements of a row are adjacent; the row pitch of an output is not below its width, that of an
 *     input may be (0: every row is the same memory);
 *   - `workspace` is caller-allocated device memory, 16-byte aligned, at least the *_workspace_bytes() of the same sizes (0 for sizes beyond
 *     an operator's limits, which the operator then refuses); it holds nothing between calls.  Two calls that may run at the same time (two streams, two captured graphs) need a workspace each;
 *   - an output overlaps no input and no other output, except where it is said to.
 * Every operator may be captured into a graph (kernel launches only) and gives the same bits on every call.
 */
#ifndef ENVIDR_BLOCKS_H
#define ENVIDR_BLOCKS_H

#include "envidr_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { ENVIDR_F32 = 0, ENVIDR_BF16 = 1, ENVIDR_F16 = 2 };
enum { ENVIDR_ACT_SILU = 0, ENVIDR_ACT_GELU = 1, ENVIDR_ACT_RELU = 2, ENVIDR_ACT_SIGMOID = 3 };   /* GELU: the tanh form */

/* version of this header: bumped on any signature change and when entry points are added */
int envidr_blocks_abi_version(void);

/* ------------------------------------------------------------------------------------------
 * gated feed-forward block
 *   g = x Wg^T, u = x Wu^T, h = act(g) * u, y = h Wd^T
 *   x [M, D], Wg / Wu [F, D], Wd [O, F], y [M, O].  D, F, O >= 1 of any remainder; 16-bit types: fastest where widths and pitches are
 *   multiples of 8 and the tensors 16-byte aligned.
 * Arithmetic.  16-bit types: products on the 16-bit matrix cores, accumulated in fp32; h (forward) and dg, du, h (backward) are rounded
 * to the type once, as the next product's operands.  fp32: every operand is carried as three bf16 terms (24 significant bits; of
 * numbers below 2^-108 what is above 2^-126), the six products above 2^-24 are accumulated in fp32; an infinity in an operand gives NaN.  Up to 32 rows (fp32: 64) go forward through a
 * kernel that streams the weights once (fp32: on the fp32 matrix cores) and keeps h in 32 bits.  fp16: a hidden unit above 65504 is an infinity.
 * Limits: D, F, O <= 2^20, F D and O F <= 2^32, M < 2^31 - 256, row pitches <= 2^21.
 * backward: dx [M, D], dw_gate / dw_up [F, D], dw_down [O, F] (any of them may be NULL: not computed).  It needs x, dy and the weights
 * only: g and u are formed again.
 * ------------------------------------------------------------------------------------------ */
uint64_t envidr_gated_mlp_workspace_bytes(uint32_t M, uint32_t D, uint32_t F, uint32_t O, int dtype, int backward);
int envidr_gated_mlp_forward(const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate, const void* w_up, int64_t ld_up,
                             const void* w_down, int64_t ld_down, uint32_t M, uint32_t D, uint32_t F, uint32_t O, int dtype, int activation,
                             void* y, int64_t ldy, void* workspace, uint64_t workspace_bytes, envidr_stream_t stream);
int envidr_gated_mlp_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate,
                              const void* w_up, int64_t ld_up, const void* w_down, int64_t ld_down, uint32_t M, uint32_t D, uint32_t F,
                              uint32_t O, int dtype, int activation, void* dx, int64_t lddx, void* dw_gate, void* dw_up, void* dw_down,
                              void* workspace, uint64_t workspace_bytes, envidr_stream_t stream);

/* ------------------------------------------------------------------------------------------
 * gated linear recurrence along packed rays
 *   a_t = sigmoid(gate_t);  h_t = a_t h_{t-1} + (1 - a_t) v_t   (blend != 0)   or   a_t h_{t-1} + v_t   (blend == 0)
 *   gate, value, h [T, C]; rays int32 [N, 3] = (id, offset, count) as envidr_march_rays_train writes them: rows offset .. offset + count - 1
 *   are the samples of ray `id`, front to back.  Rays may come in any order and leave rows between and behind them; no two may share a
 *   row or an id.  A ray with count <= 0, offset < 0 or offset + count > T has no rows (the compositors' rule).
 *   state fp32 [N, C] or NULL (zeros): h before the first sample, indexed by id; last fp32 [N, C]: h after the last one.  The id of a ray
 *   without rows, and an id that no ray names, keep their state; a ray with an id outside 0 .. N-1 starts from zeros and leaves none.
 *   Rows that belong to no ray: h, dgate and dvalue are zero there.  A NaN or an infinity stays with its ray and channel, and along them
 *   (an infinity is one, or NaN from a row on whose gate is below -87: its weight is 0 in 32 bits).
 *   Limits: T < 2^31, 65 N + T < 2^32 - 2^20, C <= 2^19.
 *   saved: fp32 [envidr_ray_recurrence_saved_floats(T, N, C)] or NULL; written by the forward pass and read by the backward one of the
 *   same inputs.
 * backward: dh [T, C], dlast fp32 [N, C] or NULL -> dgate, dvalue [T, C], dstate fp32 [N, C] or NULL.
 * ------------------------------------------------------------------------------------------ */
uint64_t envidr_ray_recurrence_saved_floats(uint64_t T, uint32_t N, uint32_t C);
uint64_t envidr_ray_recurrence_workspace_bytes(uint64_t T, uint32_t N, uint32_t C);
int envidr_ray_recurrence_forward(const void* gate, const void* value, const int32_t* rays, const float* state, uint64_t T, uint32_t N,
                                  uint32_t C, int dtype, int blend, void* h, float* last, float* saved, void* workspace,
                                  uint64_t workspace_bytes, envidr_stream_t stream);
int envidr_ray_recurrence_backward(const void* dh, const float* dlast, const void* gate, const void* value, const int32_t* rays,
                                   const float* state, const float* saved, uint64_t T, uint32_t N, uint32_t C, int dtype, int blend,
                                   void* dgate, void* dvalue, float* dstate, void* workspace, uint64_t workspace_bytes,
                                   envidr_stream_t stream);

/* ------------------------------------------------------------------------------------------
 * counter-based dropout
 *   y_i = residual_i + (keep_i ? x_i / (1 - q) : 0),   q = round(65536 p) / 65536,   keep_i = bits_i >= 65536 q
 *   bits_i: 16 of the 128 bits of Philox4x32-10 (Salmon et al. 2011) with key rng[0] and counter (i / 8, rng[1]), i the element's index;
 *   rng int64 [2] on the device, so a captured graph draws from whatever stands there when it is replayed.  p in [0, 1]; residual may be
 *   NULL.  The gradient is the same call on dy without a residual.  x, residual, y: n <= 2^35 - 2048 adjacent elements; y may be x or the residual.
 * envidr_dropout_step: used[0..1] = rng[0..1], then rng[1] += 1 -- a call's own copy of the generator, for its backward pass.
 * ------------------------------------------------------------------------------------------ */
int envidr_dropout(const void* x, const void* residual, const int64_t* rng, uint64_t n, double p, int dtype, void* y, envidr_stream_t stream);
int envidr_dropout_step(int64_t* rng, int64_t* used, envidr_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* ENVIDR_BLOCKS_H */
