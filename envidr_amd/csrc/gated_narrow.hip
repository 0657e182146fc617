// The gated feed-forward block of narrow layers, forward.
// The shading heads' shape (72 -> 256 -> 12): all weights fit one CU's LDS, and the hidden layer never leaves the registers.  A workgroup
// lays the weights out in LDS once; from there on each wave takes 32 rows at a time by itself, x straight into registers (the next rows'
// loads under the present ones' products), 32 hidden units after the other:
//   g, u = 2 x 2 blocks of 16 units (the four share the x operands), h = act(g) u in registers, rounded to the type;
//   a lane holds h of units 4 g' .. 4 g' + 3 of both blocks (g' = lane / 16) for its row: exactly eight k of the next product's operand, in an
//   order of k that Wd's rows in LDS follow, so y += h Wd^T needs no exchange between lanes.
// Bound: the activation on the vector ALU (two quarter-rate instructions and about eight others a hidden unit and row), then the products.
// 524 288 rows of 72 -> 256 -> 12 in fp16: 78 us; 99 991 rows 22 us (in two kernels, h through memory: 70).
#include "gated_mlp.hip.h"
#include "gemm_core.hip.h"

#include <type_traits>

namespace envidr {
namespace {

constexpr int kNarrowLds = 160 * 1024, kNarrowRows = 32;
// waves of a workgroup: sixteen where 128 registers are enough (a wave alone waits for its own chain of products and exponentials: 99991 rows of
// 72 -> 256 -> 12 take 27 us with eight), else eight
constexpr int narrow_waves(int kd, int ob) { return kd <= 3 && ob == 1 ? 16 : 8; }
constexpr uint32_t narrow_units(uint32_t kd) { return kd == 1 ? 4u : kd == 2 ? 8u : 16u; }          // 16-byte units of a weight row in LDS
__host__ __device__ inline uint32_t narrow_down_units(uint32_t hidden) { return hidden / 8u + (20u - hidden / 8u % 16u) % 16u; }      // of a row of Wd: 4 mod 16

__device__ __forceinline__ uint32_t narrow_swizzle(uint32_t units, uint32_t row) {
    const uint32_t i = row & 15u, p = units == 4u ? i >> 2 : units == 8u ? i >> 1 : i;
    return p ^ ((units == 4u ? p ^ (p >> 1) : units == 8u ? (p >> 1) ^ (p >> 2) : (p >> 2) ^ (p >> 3)) & 1u);
}

// KD: k blocks of 32 of the input width; OB: blocks of 16 of the output width
template <class E, int ACT, int KD, int OB> __global__ void __launch_bounds__(narrow_waves(KD, OB) * 64, narrow_waves(KD, OB) / 4) k_narrow_forward(NarrowArgs a) {
    constexpr int kNarrowWaves = narrow_waves(KD, OB);
    constexpr int MI = kNarrowRows / 16;
    constexpr uint32_t kUnits = narrow_units(KD);
    __shared__ __attribute__((aligned(1024))) char lds_all[kNarrowLds];
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_void*)lds_all, lane = threadIdx.x & 63u, g = lane >> 4, i = lane & 15u;
    const uint32_t hidden = (a.F + 31u) / 32u * 32u, down = lds + 2u * hidden * kUnits * 16u, down_units = narrow_down_units(hidden);
    const E *wg = static_cast<const E*>(a.wg), *wu = static_cast<const E*>(a.wu), *wd = static_cast<const E*>(a.wd);
    const bool whole = a.D % 8u == 0u;
    const uint32_t tiles = (a.M + kNarrowRows - 1u) / kNarrowRows, by = gridDim.x * kNarrowWaves;
    // (tile t is wave t / gridDim's of workgroup t % gridDim: what is left of a round is spread over all CUs)
    uint32_t t = (threadIdx.x >> 6) * gridDim.x + blockIdx.x;
    struct Rows {
        s16x8 x[MI][KD];
    } now, next;
    auto fetch = [&](Rows& r, uint32_t t) {
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
            const E* row = static_cast<const E*>(a.x) + (int64_t)min(t * kNarrowRows + mi * 16u + i, a.M - 1u) * a.ldx;
#pragma unroll
            for (int kk = 0; kk < KD; ++kk) r.x[mi][kk] = load8(row, kk * 32u + g * 8u, a.D, whole);
        }
    };
    if (t < tiles) fetch(now, t);
    // weights: blocks of 16 rows, per 32 hidden units gate, gate, up, up; a batch's loads before its stores
    constexpr uint32_t kThreads = kNarrowWaves * 64, kBatch = 6;
    for (uint32_t first = threadIdx.x; first < 2u * hidden * (KD * 4u); first += kBatch * kThreads) {
        s16x8 v[kBatch];
        uint32_t to[kBatch];
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            const uint32_t at = min(first + b * kThreads, 2u * hidden * (KD * 4u) - 1u), row = at / (KD * 4u), unit = at % (KD * 4u), f = (row >> 6) * 32u + (row & 31u), fc = min(f, a.F - 1u);
            v[b] = load8(row & 32u ? wu + (int64_t)fc * a.lu : wg + (int64_t)fc * a.lg, unit * 8u, a.D, whole);
            if (f >= a.F) v[b] = s16x8{};
            to[b] = lds + (row * kUnits + (unit ^ narrow_swizzle(kUnits, row))) * 16u;
        }
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) *(lds_s16x8*)to[b] = v[b];         // (past the end: the last unit again)
    }
    for (uint32_t at = threadIdx.x; at < OB * 16u * (hidden / 8u); at += kNarrowWaves * 64) {
        const uint32_t o = at / (hidden / 8u), unit = at % (hidden / 8u), f = unit / 4u * 32u + 4u * (unit % 4u);
        Pack<E, 8> v;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const uint32_t k = f + (j < 4 ? j : 12u + j);
            v.v[j] = o < a.O && k < a.F ? wd[(int64_t)o * a.ldn + k] : from_f32<E>(0.0f);
        }
        *(lds_s16x8*)(down + (o * down_units + (unit ^ narrow_swizzle(4u, o))) * 16u) = __builtin_bit_cast(s16x8, v);
    }
    __syncthreads();
    auto work = [&](const Rows& r, uint32_t t) {
        f32x4 y[MI][OB] = {};
        for (uint32_t hb = 0; hb < hidden / 32u; ++hb) {
            f32x4 p[MI][4] = {};
#pragma unroll
            for (int kk = 0; kk < KD; ++kk)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const s16x8 w = *(const lds_s16x8*)(lds + ((hb * 64u + b * 16u + i) * kUnits + ((kk * 4u + g) ^ narrow_swizzle(kUnits, i))) * 16u);
#pragma unroll
                    for (int mi = 0; mi < MI; ++mi) p[mi][b] = mfma16<E>(w, r.x[mi][kk], p[mi][b]);
                }
            s16x8 h[MI];
#pragma unroll
            for (int mi = 0; mi < MI; ++mi) {
                Pack<E, 8> v;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        v.v[4 * b + q] = from_f32<E>(activation_value<ACT, false>(p[mi][b][q]) * p[mi][b + 2][q]);
                    }
                // (units behind the last one: weights of zero, which an infinity in x makes NaN)
                if (hb * 32u + 32u > a.F) {
#pragma unroll
                    for (int n = 0; n < 8; ++n)
                        if (hb * 32u + 16u * (n >> 2) + 4u * g + (n & 3) >= a.F) v.v[n] = from_f32<E>(0.0f);
                }
                h[mi] = __builtin_bit_cast(s16x8, v);
            }
#pragma unroll
            for (int ob = 0; ob < OB; ++ob) {
                const s16x8 w = *(const lds_s16x8*)(down + ((ob * 16u + i) * down_units + ((hb * 4u + g) ^ narrow_swizzle(4u, i))) * 16u);
#pragma unroll
                for (int mi = 0; mi < MI; ++mi) y[mi][ob] = mfma16<E>(w, h[mi], y[mi][ob]);
            }
        }
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
            const uint32_t m = t * kNarrowRows + mi * 16u + i;
            if (m >= a.M) continue;
#pragma unroll
            for (int ob = 0; ob < OB; ++ob) {
                const uint32_t n = ob * 16u + 4u * g;
                const float v[4] = {y[mi][ob][0], y[mi][ob][1], y[mi][ob][2], y[mi][ob][3]};
                store_row4(static_cast<E*>(a.y) + (int64_t)m * a.ldy + n, (int64_t)a.O - n, v);
            }
        }
    };
    if (t >= tiles) return;
    for (;;) {
        if (t + by < tiles) fetch(next, t + by);
        work(now, t);
        if ((t += by) >= tiles) return;
        if (t + by < tiles) fetch(now, t + by);
        work(next, t);
        if ((t += by) >= tiles) return;
    }
}

template <class E, int ACT> int launch_narrow(const NarrowArgs& a, hipStream_t s) {
    const uint32_t tiles = ceil_div(a.M, (uint32_t)kNarrowRows), grid = tiles < 256u ? tiles : 256u;
    auto go = [&](auto kd, auto ob) { hipLaunchKernelGGL((k_narrow_forward<E, ACT, decltype(kd)::value, decltype(ob)::value>), dim3(grid), dim3(narrow_waves(decltype(kd)::value, decltype(ob)::value) * 64), 0, s, a); };
    auto with_kd = [&](auto kd) {
        if (a.O <= 16) go(kd, std::integral_constant<int, 1>{});
        else go(kd, std::integral_constant<int, 4>{});
    };
    switch (ceil_div(a.D, 32u)) {
        case 1: with_kd(std::integral_constant<int, 1>{}); break;
        case 2: with_kd(std::integral_constant<int, 2>{}); break;
        case 3: with_kd(std::integral_constant<int, 3>{}); break;
        default: with_kd(std::integral_constant<int, 4>{}); break;
    }
    return check_launch("k_narrow_forward");
}

}  // namespace

bool gated_is_narrow(uint32_t D, uint32_t F, uint32_t O, int dtype) {
    if (dtype == ENVIDR_F32) return D <= 96 && F <= 256 && O <= 32;              // (the weights' three terms in eight waves' registers)
    if (D > 128 || O > 64 || F > 4096) return false;
    const uint32_t hidden = (F + 31u) / 32u * 32u;
    return 2u * hidden * narrow_units((D + 31u) / 32u) * 16u + (O <= 16u ? 16u : 64u) * narrow_down_units(hidden) * 16u <= (uint32_t)kNarrowLds;
}

int gated_narrow_forward(const NarrowArgs& a, int dtype, int activation, hipStream_t s) {
    if (dtype == ENVIDR_F32) return gated_narrow_forward_fp32(a, activation, s);
    if (dtype == ENVIDR_BF16) ENVIDR_FOR_ACT(activation, ACT, return (launch_narrow<__bf16, ACT>(a, s)));
    ENVIDR_FOR_ACT(activation, ACT, return (launch_narrow<_Float16, ACT>(a, s)));
}

}  // namespace envidr
