// Shared by the sources of the gated feed-forward block.
#pragma once
#include "blocks_common.hip.h"

namespace envidr {

#define ENVIDR_FOR_ACT(act, ACT, ...)                                                                  \
    do {                                                                                               \
        if ((act) == ENVIDR_ACT_SILU) { constexpr int ACT = ENVIDR_ACT_SILU; __VA_ARGS__; }            \
        else if ((act) == ENVIDR_ACT_GELU) { constexpr int ACT = ENVIDR_ACT_GELU; __VA_ARGS__; }       \
        else if ((act) == ENVIDR_ACT_RELU) { constexpr int ACT = ENVIDR_ACT_RELU; __VA_ARGS__; }       \
        else { constexpr int ACT = ENVIDR_ACT_SIGMOID; __VA_ARGS__; }                                  \
    } while (0)

// a whole forward pass: row pitches in elements, any alignment
struct NarrowArgs {
    const void *x, *wg, *wu, *wd;
    void* y;
    int64_t ldx, lg, lu, ldn, ldy;
    uint32_t M, D, F, O;
};

// widths whose weights fit one CU's LDS (fp32: registers), and their forward pass
bool gated_is_narrow(uint32_t D, uint32_t F, uint32_t O, int dtype);
int gated_narrow_forward(const NarrowArgs& a, int dtype, int activation, hipStream_t s);

// The kernels whose waves share rows in teams: waves that take a team's rows together, 32 hidden units each: a power of two; all eight of them from
// 65 input columns on, where several teams' rows on their way do not fit the registers.
constexpr uint32_t kTeamWaves = 8;
__host__ __device__ inline uint32_t narrow_slices(uint32_t D, uint32_t F) { return D > 64u || F > 128u ? 8u : F > 64u ? 4u : F > 32u ? 2u : 1u; }

// fp32 forward, D <= 96, F <= 256, O <= 32
int gated_narrow_forward_fp32(const NarrowArgs& a, int activation, hipStream_t s);

// gradients of the 16-bit types: dx [M][D] or NULL; the weights' as `parts` partial sums in fp32, part = [parts][F][D] of the gate, the same of the up, [parts][O][F] of
// the down matrix
struct NarrowGradArgs {
    const void *dy, *x, *wg, *wu, *wd;
    void* dx;
    float* part;
    int64_t lddy, ldx, lg, lu, ldn, lddx;
    uint32_t M, D, F, O, slices;    // slices: set by the launch
    bool want_w;
};
bool gated_grad_is_narrow(uint32_t D, uint32_t F, uint32_t O, int dtype);
uint32_t gated_narrow_grad_parts(uint32_t M, uint32_t D, uint32_t F);
int gated_narrow_backward(NarrowGradArgs a, int dtype, int activation, hipStream_t s);

}  // namespace envidr
