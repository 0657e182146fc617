// Counter-based dropout: y_i = residual_i + keep_i x_i / (1 - q).  keep_i is a pure function of (rng, i), so the backward pass computes it
// again and no mask is stored.
//
// Generator: Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011): ten rounds of two 32 x 32
// -> 64 bit products.  One call gives 128 bits = eight elements of 16 bits: drop probabilities are multiples of 2^-16, which no training run
// can tell from the asked one, and 1 / (1 - q) uses the multiple, so the expectation is exact.  With 32 bits an element (four a call) the
// products alone would cost more than the memory: twenty 64-bit products a call, a quarter-rate instruction each.
// Bound: memory.  A thread owns eight elements: 16 bytes a stream in the 16-bit types, 32 in fp32.
#include "blocks_common.hip.h"

namespace envidr {
namespace {

struct Philox {
    uint32_t w[4];
};

__device__ __forceinline__ Philox philox10(uint64_t key, uint64_t lo, uint64_t hi) {
    uint32_t c0 = (uint32_t)lo, c1 = (uint32_t)(lo >> 32), c2 = (uint32_t)hi, c3 = (uint32_t)(hi >> 32);
    uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p = (uint64_t)c0 * 0xD2511F53u, q = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(q >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)q;
        c2 = (uint32_t)(p >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

template <class E, bool RES>
__global__ void __launch_bounds__(kBlock) k_dropout(const E* x, const E* residual, const int64_t* __restrict__ rng, uint64_t n, uint32_t limit, float scale,
                                                    E* y) {
    const uint64_t unit = (uint64_t)blockIdx.x * kBlock + threadIdx.x, first = unit * 8;
    if (first >= n) return;
    const Philox z = philox10((uint64_t)rng[0], unit, (uint64_t)rng[1]);
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = ((z.w[j >> 1] >> (16 * (j & 1))) & 0xFFFFu) >= limit ? scale : 0.0f;
    if (first + 8 <= n) {
        const Pack<E, 8> vx = load_pack<E, 8>(x + first);
        Pack<E, 8> vr, out;
        if constexpr (RES) vr = load_pack<E, 8>(residual + first);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // (a dropped element is 0 whatever x holds: 0 * inf would be NaN)
            const float v = f[j] != 0.0f ? to_f32(vx.v[j]) * f[j] : 0.0f;
            out.v[j] = from_f32<E>(RES ? v + to_f32(vr.v[j]) : v);
        }
        store_pack(y + first, out);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (first + j >= n) break;
            const float v = f[j] != 0.0f ? to_f32(x[first + j]) * f[j] : 0.0f;
            y[first + j] = from_f32<E>(RES ? v + to_f32(residual[first + j]) : v);
        }
    }
}

__global__ void k_dropout_step(int64_t* rng, int64_t* used) {
    if (threadIdx.x == 0 && blockIdx.x == 0) {
        const int64_t key = rng[0], call = rng[1];
        used[0] = key;
        used[1] = call;
        rng[1] = (int64_t)((uint64_t)call + 1u);
    }
}

}  // namespace
}  // namespace envidr

using namespace envidr;

extern "C" {

int envidr_blocks_abi_version(void) { return 1; }

int envidr_dropout(const void* x, const void* residual, const int64_t* rng, uint64_t n, double p, int dtype, void* y, envidr_stream_t stream) {
    ENVIDR_REQUIRE(dtype_ok(dtype), "dropout: unknown dtype %d", dtype);
    ENVIDR_REQUIRE(p >= 0.0 && p <= 1.0, "dropout: p=%g is not a probability", p);
    if (n == 0) return ENVIDR_OK;
    ENVIDR_REQUIRE(x && rng && y, "dropout: null pointer");
    // (a launch holds fewer than 2^32 threads)
    ENVIDR_REQUIRE(n <= (1ull << 35) - 8ull * kBlock, "dropout: %llu elements are too many for one call", (unsigned long long)n);
    const uint64_t blocks = (n + 8ull * kBlock - 1) / (8ull * kBlock);
    const uint32_t limit = (uint32_t)__builtin_rint(p * 65536.0);
    const float scale = limit >= 65536u ? 0.0f : (float)(65536.0 / (65536.0 - (double)limit));
    hipStream_t s = as_stream(stream);
    ENVIDR_FOR_DTYPE(dtype, E, {
        const E* xe = static_cast<const E*>(x);
        const E* re = static_cast<const E*>(residual);
        if (re) hipLaunchKernelGGL((k_dropout<E, true>), dim3((uint32_t)blocks), dim3(kBlock), 0, s, xe, re, rng, n, limit, scale, static_cast<E*>(y));
        else hipLaunchKernelGGL((k_dropout<E, false>), dim3((uint32_t)blocks), dim3(kBlock), 0, s, xe, re, rng, n, limit, scale, static_cast<E*>(y));
    });
    return check_launch("k_dropout");
}

int envidr_dropout_step(int64_t* rng, int64_t* used, envidr_stream_t stream) {
    ENVIDR_REQUIRE(rng && used, "dropout_step: null pointer");
    hipLaunchKernelGGL(k_dropout_step, dim3(1), dim3(64), 0, as_stream(stream), rng, used);
    return check_launch("k_dropout_step");
}

}  // extern "C"
