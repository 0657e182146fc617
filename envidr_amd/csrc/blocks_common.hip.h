// Shared by the block operators (include/envidr_blocks.h): element types, vector loads / stores of any alignment, activations.
#pragma once
#include "common.hip.h"
#include "../../include/envidr_blocks.h"

namespace envidr {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <class E> __device__ __forceinline__ float to_f32(E v) { return (float)v; }
template <class E> __device__ __forceinline__ E from_f32(float v) { return (E)v; }             // round to nearest even, NaN stays NaN

// N adjacent elements as one memory operation; the address needs the element's own alignment only (global accesses of any alignment are
// legal on gfx950, they cost an extra request where a line ends inside)
template <class E, int N> struct __attribute__((packed, aligned(sizeof(E)))) Pack { E v[N]; };
template <class E, int N> __device__ __forceinline__ Pack<E, N> load_pack(const E* p) { return *reinterpret_cast<const Pack<E, N>*>(p); }
template <class E, int N> __device__ __forceinline__ void store_pack(E* p, const Pack<E, N>& v) { *reinterpret_cast<Pack<E, N>*>(p) = v; }

// sigmoid(v) and sigmoid(-v), both to full relative precision at either end (1 - sigmoid would lose it where sigmoid -> 1), from one
// exponential e = 2^(-|v| log2 e).  FINE: the product's rounding puts an error of |v| 2^-24 on e -- nothing beside the steps of 16-bit inputs
// and results; fp32 takes the product's low part along.
template <bool FINE> __device__ __forceinline__ void sigmoid_pair(float v, float& s, float& s_neg) {
    float x = fabsf(v), e;
    if constexpr (FINE) {
        x = x > 150.0f ? 150.0f : x;                 // (e is 0 there; an infinity would make the low part NaN)
        const float t = x * -1.44269504f, lo = fmaf(x, -1.44269504f, -t) - x * 1.92596299e-8f;
        e = __builtin_amdgcn_exp2f(t);
        e = fmaf(e, lo * 0.693147181f, e);
    } else {
        e = __builtin_amdgcn_exp2f(x * -1.44269504f);
    }
    const float r = __builtin_amdgcn_rcpf(1.0f + e), er = e * r;
    s = v < 0.0f ? er : r;
    s_neg = v < 0.0f ? r : er;                       // (a NaN: e, and so both)
}

// act(g) and act'(g)
template <int ACT, bool FINE> __device__ __forceinline__ void activation(float g, float& a, float& da) {
    if constexpr (ACT == ENVIDR_ACT_RELU) {
        a = g < 0.0f ? 0.0f : g;                 // (NaN stays NaN)
        da = g > 0.0f ? 1.0f : 0.0f;
    } else if constexpr (ACT == ENVIDR_ACT_SIGMOID) {
        float sn;
        sigmoid_pair<FINE>(g, a, sn);
        da = a * sn;
    } else if constexpr (ACT == ENVIDR_ACT_SILU) {
        float s, sn;
        sigmoid_pair<FINE>(g, s, sn);
        a = g * s;
        da = fmaf(a, sn, s);
    } else {
        // 0.5 g (1 + tanh z) = g sigmoid(2 z), z = sqrt(2 / pi) (g + 0.044715 g^3); beyond |g| = 16 the sigmoid is 0 or 1 to the last bit
        const float k2 = 1.5957691216057308f, c = 0.044715f;
        const float cg = g > 16.0f ? 16.0f : (g < -16.0f ? -16.0f : g), q = cg * cg;
        float s, sn;
        sigmoid_pair<FINE>(k2 * cg * fmaf(c, q, 1.0f), s, sn);
        a = g * s;
        da = fmaf(cg * s * sn, k2 * fmaf(3.0f * c, q, 1.0f), s);
    }
}

// act(g) alone (forward).  For 16-bit results the one-sided sigmoid 1 / (1 + 2^(-v log2 e)) does: it overflows to 0 where it should.
template <int ACT, bool FINE> __device__ __forceinline__ float activation_value(float g) {
    if constexpr (FINE || ACT == ENVIDR_ACT_RELU) {
        float a, da;
        activation<ACT, FINE>(g, a, da);
        return a;
    } else {
        float z = g;
        if constexpr (ACT == ENVIDR_ACT_GELU) z = 1.5957691216057308f * g * fmaf(0.044715f, g * g, 1.0f);
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f));
        return ACT == ENVIDR_ACT_SIGMOID ? s : g * s;
    }
}

#define ENVIDR_FOR_DTYPE(dtype, E, ...)                                  \
    do {                                                                 \
        if ((dtype) == ENVIDR_F32) { using E = float; __VA_ARGS__; }     \
        else if ((dtype) == ENVIDR_BF16) { using E = __bf16; __VA_ARGS__; } \
        else { using E = _Float16; __VA_ARGS__; }                        \
    } while (0)

static inline bool dtype_ok(int d) { return d == ENVIDR_F32 || d == ENVIDR_BF16 || d == ENVIDR_F16; }
static inline uint32_t dtype_size(int d) { return d == ENVIDR_F32 ? 4u : 2u; }
static inline uint64_t round_up64(uint64_t v, uint64_t to) { return (v + to - 1) / to * to; }

}  // namespace envidr
