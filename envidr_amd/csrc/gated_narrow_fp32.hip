// The gated feed-forward block of narrow layers in fp32, forward, in one kernel: the weights stay in registers, the hidden layer too.
//
// A workgroup's eight waves form teams of `slices` waves; a team takes 32 rows at a time, a wave 32 hidden units of them.  The wave keeps its units'
// weights, gate, up and down, as their three bf16 terms each (3 x 2 x 24 + 24 registers at 96 input columns); x comes from LDS, whose rows the
// workgroup splits into terms once for all its waves.  g and u from the six products of the terms, h = act(g) u in 32 bits, split again: a lane
// holds units 4 q .. 4 q + 3 and 16 + 4 q .. 16 + 4 q + 3 of its row (q = lane / 16), which is one operand of the second product, in an order of k
// that the lanes' parts of Wd follow.  So a wave forms its units' share of y by itself; the shares meet in LDS and are added up in the order of the
// units.
// Bound: matrix cores (six products a product: about 45 % of the time) and vector ALU (activation, terms of h: 40 %), which the two waves of a SIMD
// use in turns.  146 000 rows of 72 -> 256 -> 12: 104 us by itself, 119 behind a backward pass, whose operands have taken x's place in the caches (operands
// laid out and the hidden layer through memory: 232); of 32 -> 64 -> 16 30 (71); 65 rows 18 (30).
#include "gated_mlp.hip.h"
#include "gemm_core.hip.h"

#include <type_traits>

namespace envidr {
namespace {

constexpr int kLds = 160 * 1024, kWaves = kTeamWaves, kTeamRows = 32, kOut = 2;          // kOut: blocks of 16 output columns

struct Terms8 {
    s16x8 t[3];
};
__device__ __forceinline__ Terms8 split8(const float (&v)[8]) {
    Pack<__bf16, 8> o[3];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        __bf16 t[3];
        split3(v[i], t);
#pragma unroll
        for (int p = 0; p < 3; ++p) o[p].v[i] = t[p];
    }
    return {{__builtin_bit_cast(s16x8, o[0]), __builtin_bit_cast(s16x8, o[1]), __builtin_bit_cast(s16x8, o[2])}};
}
// eight adjacent elements from column k of a row of n, zeros behind it
struct Floats8 {
    float v[8];
};
__device__ __forceinline__ Floats8 floats8(const float* row, uint32_t k, uint32_t n) {
    Floats8 r;
    if (k + 8u <= n) {
        const Pack<float, 4> a = load_pack<float, 4>(row + k), b = load_pack<float, 4>(row + k + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { r.v[i] = a.v[i]; r.v[4 + i] = b.v[i]; }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) r.v[i] = k + i < n ? row[k + i] : 0.0f;
    }
    return r;
}
// c += w x, the small products first
__device__ __forceinline__ f32x4 six(const Terms8& w, const Terms8& x, f32x4 c) {
    c = mfma16<__bf16>(w.t[2], x.t[0], c);
    c = mfma16<__bf16>(w.t[0], x.t[2], c);
    c = mfma16<__bf16>(w.t[1], x.t[1], c);
    c = mfma16<__bf16>(w.t[1], x.t[0], c);
    c = mfma16<__bf16>(w.t[0], x.t[1], c);
    return mfma16<__bf16>(w.t[0], x.t[0], c);
}

// KD: k blocks of 32 of the input width; ONE: one team, whose rows are one unit of eight a thread at most
template <int ACT, int KD, bool ONE> __global__ void __launch_bounds__(kWaves * 64, 2) k_narrow_forward_fp32(NarrowArgs a) {
    constexpr uint32_t kXPitch = KD * 64 + 32, kPlane = kTeamRows * kXPitch, kTeamBytes = 3 * kPlane;
    constexpr int kXUnits = ONE ? 1 : 2 * KD;
    __shared__ __attribute__((aligned(1024))) char lds_all[kLds];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, i = lane & 15u;
    const uint32_t slices = ONE ? kWaves : narrow_slices(a.D, a.F), team = ONE ? 0u : wave / slices, slice = ONE ? wave : wave % slices, teams = kWaves / slices;
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_void*)lds_all, xs = lds + kWaves * (4u * kOut * 512u), x_mine = xs + team * kTeamBytes;
    const float *wg = static_cast<const float*>(a.wg), *wu = static_cast<const float*>(a.wu), *wd = static_cast<const float*>(a.wd);
    const uint32_t rows = teams * kTeamRows, tiles = (a.M + rows - 1u) / rows;
    Floats8 nx[kXUnits];
    auto fetch = [&](uint32_t t) {
#pragma unroll
        for (int j = 0; j < kXUnits; ++j) {
            const uint32_t n = j * (kWaves * 64u) + threadIdx.x, r = n / (KD * 4u), m = t * rows + r;
            if (r < rows) nx[j] = floats8(static_cast<const float*>(a.x) + (int64_t)min(m, a.M - 1u) * a.ldx, n % (KD * 4u) * 8u, a.D);
        }
    };
    auto put = [&] {
#pragma unroll
        for (int j = 0; j < kXUnits; ++j) {
            const uint32_t n = j * (kWaves * 64u) + threadIdx.x, r = n / (KD * 4u);
            if (r >= rows) continue;
            const Terms8 s = split8(nx[j].v);
            const uint32_t at = xs + r / kTeamRows * kTeamBytes + r % kTeamRows * kXPitch + n % (KD * 4u) * 16u;
#pragma unroll
            for (int p = 0; p < 3; ++p) *(lds_s16x8*)(at + p * kPlane) = s.t[p];
        }
    };
    uint32_t t = blockIdx.x;                                     // (the grid has no more workgroups than tiles)
    fetch(t);
    Terms8 rg[2][KD], ru[2][KD], rd[kOut];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const uint32_t f = slice * 32u + b * 16u + i, fc = min(f, a.F - 1u), n = f < a.F ? a.D : 0u;
#pragma unroll
        for (int kk = 0; kk < KD; ++kk) {
            rg[b][kk] = split8(floats8(wg + (int64_t)fc * a.lg, kk * 32u + g * 8u, n).v);
            ru[b][kk] = split8(floats8(wu + (int64_t)fc * a.lu, kk * 32u + g * 8u, n).v);
        }
    }
#pragma unroll
    for (int o = 0; o < kOut; ++o) {
        float v[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const uint32_t f = slice * 32u + (j < 4 ? 0u : 16u) + 4u * g + (j & 3u), n = o * 16u + i;
            v[j] = f < a.F && n < a.O ? wd[(int64_t)n * a.ldn + f] : 0.0f;
        }
        rd[o] = split8(v);
    }
    put();
    lds_barrier();
    for (;;) {
        const bool more = t + gridDim.x < tiles;
        if (more) fetch(t + gridDim.x);
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
            f32x4 pg[2] = {}, pu[2] = {};
#pragma unroll
            for (int kk = 0; kk < KD; ++kk) {
                Terms8 x;
#pragma unroll
                for (int p = 0; p < 3; ++p) x.t[p] = *(const lds_s16x8*)(x_mine + p * kPlane + (rb * 16u + i) * kXPitch + (kk * 4u + g) * 16u);
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    pg[b] = six(rg[b][kk], x, pg[b]);
                    pu[b] = six(ru[b][kk], x, pu[b]);
                }
            }
            float h[8];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int q = 0; q < 4; ++q) h[4 * b + q] = activation_value<ACT, true>(pg[b][q]) * pu[b][q];
            const Terms8 s = split8(h);
#pragma unroll
            for (int o = 0; o < kOut; ++o)
                if (o == 0 || a.O > 16u) *(lds_f32x4*)(lds + ((wave * 2u + rb) * kOut + o) * 1024u + lane * 16u) = six(rd[o], s, f32x4{});
        }
        lds_barrier();
        // the shares: unit n is (team, rows, columns, lane)'s four columns
        for (uint32_t n = threadIdx.x; n < teams * (2u * kOut * 64u); n += kWaves * 64u) {
            const uint32_t part = n / 64u % (2u * kOut), of = n / (2u * kOut * 64u);
            f32x4 s = {};
            for (uint32_t k = 0; k < slices; ++k) s += *(const lds_f32x4*)(lds + ((of * slices + k) * (2u * kOut) + part) * 1024u + lane * 16u);
            const uint32_t m = t * rows + of * kTeamRows + part / kOut * 16u + i, c = part % kOut * 16u + 4u * g;
            if (m >= a.M || c >= a.O) continue;
            const float v[4] = {s[0], s[1], s[2], s[3]};
            store_row4(static_cast<float*>(a.y) + (int64_t)m * a.ldy + c, (int64_t)a.O - c, v);
        }
        if (!more) return;
        put();
        lds_barrier();
        t += gridDim.x;
    }
}

template <int ACT> int launch(const NarrowArgs& a, uint32_t grid, bool one, hipStream_t s) {
    auto go = [&](auto kd, auto o) { hipLaunchKernelGGL((k_narrow_forward_fp32<ACT, decltype(kd)::value, decltype(o)::value>), dim3(grid), dim3(kWaves * 64), 0, s, a); };
    auto any = [&](auto kd) {
        if (one) go(kd, std::true_type{});
        else go(kd, std::false_type{});
    };
    if (a.D <= 32u) any(std::integral_constant<int, 1>{});
    else if (a.D <= 64u) any(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 3>{}, std::true_type{});
    return check_launch("k_narrow_forward_fp32");
}

}  // namespace

int gated_narrow_forward_fp32(const NarrowArgs& a, int activation, hipStream_t s) {
    const uint32_t slices = narrow_slices(a.D, a.F), tiles = ceil_div(a.M, kWaves / slices * (uint32_t)kTeamRows);
    ENVIDR_FOR_ACT(activation, ACT, return (launch<ACT>(a, tiles < 256u ? tiles : 256u, slices == kWaves, s)));
}

}  // namespace envidr
