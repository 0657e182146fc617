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

// widths whose weights fit one CU's LDS (16-bit types), and their forward pass
bool gated_is_narrow(uint32_t D, uint32_t F, uint32_t O, int dtype);
int gated_narrow_forward(const NarrowArgs& a, int dtype, int activation, hipStream_t s);

}  // namespace envidr
