// The matrix-product core of the gated feed-forward block: C[m][n] = sum_k A(m, k) B(n, k) on the 16-bit matrix cores
// (v_mfma_f32_16x16x32_{bf16,f16}, fp32 accumulators), operands given as NP planes of 16-bit terms: NP = 1 for the 16-bit types; NP = 3
// for fp32, x = x0 + x1 + x2 with bf16 terms (8 significant bits each, so the three hold all 24), of whose nine products the six above
// 2^-24 are formed: x0 y0, x0 y1, x1 y0, x1 y1, x0 y2, x2 y0.  Six bf16 products cost 6/16 of one fp32 product on this chip's matrix cores.
//
// Either operand lies in memory in one of two ways: K-CONTIGUOUS (element (r, k) at r ld + k: x W^T) or K-STRIDED (element (r, k) at
// k ld + r: the transposed factors of the gradients).  Both reach LDS by direct loads (16 bytes a lane, no registers), in memory's own order:
//   K-contiguous tile: row r = 2 KT bytes; a lane's operand (8 consecutive k) is one 16-byte read;
//   K-strided tile:    row k = 2 TR bytes; the operand is two transposing reads (ds_read_b64_tr_b16: sixteen lanes read four k rows of
//                      sixteen columns and each receives one column's four values).
// A direct load writes its 64 x 16 bytes in lane order, so the LDS layout is permuted by permuting which 16 bytes a lane FETCHES:
// within a row the unit c sits at c ^ f(row), f chosen so that the rows one read touches together fall on different banks (256 bytes).
// Edges: a 16-byte unit is wholly inside or outside (extents along the contiguous index are multiples of 8, the packing pads with zeros);
// outside units are sent past the buffer's bound, where a load delivers zeros.
#pragma once
#include "blocks_common.hip.h"

namespace envidr {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

struct Operand {
    const uint16_t* p;      // plane 0
    uint64_t plane;         // elements between planes
    uint32_t ld;            // elements between rows (K-strided: between k)
    uint32_t ext;           // rows of the operand (K-strided: a multiple of 8)
};

constexpr uint32_t kOutside = 0x80000000u;      // a buffer offset past every bound

template <class T> __device__ __forceinline__ f32x4 mfma16(s16x8 a, s16x8 b, f32x4 c) {
    if constexpr (__is_same(T, _Float16))
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// One operand's tile: TR rows x KT k, NP planes.  PAIR: the tile's rows alternate in blocks of 16 between two K-contiguous operands of
// the same shape, each with its own pitch (gate and up weights of the same hidden units land in the same wave).
template <int TR, int KT, int NP, bool KC, int WAVES, bool PAIR = false> struct TileLoad {
    static constexpr int kPlaneBytes = TR * KT * 2;
    static constexpr int kBytes = kPlaneBytes * NP;
    static constexpr int kPerPlane = kPlaneBytes / 1024;                 // wave loads of 64 x 16 bytes
    static constexpr int kLoads = kPerPlane * NP;
    static constexpr int U = (kLoads + WAVES - 1) / WAVES;
    static constexpr int kUnits = KC ? KT / 8 : TR / 8;                  // 16-byte units of an LDS row
    static_assert(kPlaneBytes % 1024 == 0 && (!PAIR || KC), "whole wave loads");

    const uint16_t* base[PAIR ? 2 : 1];
    uint64_t plane;
    uint32_t ld;
    uint32_t off[U];        // byte offset of the lane's unit from the k-step's base
    uint32_t kpos[U];       // first k of the lane's unit inside the step

    // the unit that a row holds at place s, as (row & its swizzle) -- its own inverse
    static __device__ __forceinline__ uint32_t unit_at(uint32_t row, uint32_t s) {
        if constexpr (KC) return s ^ ((row / (16u / kUnits)) & (kUnits - 1u));
        else return s ^ (2u * strided_swizzle(row));
    }
    static __device__ __forceinline__ uint32_t strided_swizzle(uint32_t k) {
        if constexpr (TR >= 128) return (k & 3u) | ((k >> 1) & 4u);
        else if constexpr (TR == 64) return ((k >> 1) & 1u) | ((k >> 2) & 2u);
        else return (k >> 3) & 1u;
    }

    __device__ __forceinline__ void init(const Operand& a, const Operand& a2, uint32_t row0, uint32_t wave, uint32_t lane) {
        plane = a.plane;
        ld = a.ld;
        base[0] = a.p + (KC ? (uint64_t)row0 * a.ld : (uint64_t)row0);
        if constexpr (PAIR) base[1] = a2.p + (uint64_t)row0 * a2.ld;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t q = wave * U + u, idx = (q % kPerPlane) * 64u + lane, r = idx / kUnits, c = unit_at(r, idx % kUnits);
            if constexpr (KC) {
                const uint32_t row = PAIR ? (r >> 5) * 16u + (r & 15u) : r, pitch = PAIR && ((r >> 4) & 1u) ? a2.ld : a.ld;
                off[u] = row0 + row < a.ext ? (row * pitch + c * 8u) * 2u : kOutside;
                kpos[u] = c * 8u;
            } else {
                off[u] = row0 + c * 8u < a.ext ? (r * a.ld + c * 8u) * 2u : kOutside;
                kpos[u] = r;
            }
        }
    }
    // starts the loads of the step that begins at k0 (of K) into `lds`
    __device__ __forceinline__ void issue(char* lds, uint32_t k0, uint32_t K, uint32_t wave) const {
        const uint64_t at = KC ? (uint64_t)k0 : (uint64_t)k0 * ld;
        const bool tail = k0 + KT > K;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint32_t q = wave * U + u;
            if (kLoads % WAVES != 0 && q >= (uint32_t)kLoads) break;
            const uint32_t pl = q / kPerPlane, in_plane = q % kPerPlane;
            const uint16_t* b = base[0];
            if constexpr (PAIR) b = (in_plane * 64u / kUnits >> 4) & 1u ? base[1] : base[0];
            b += (NP > 1 ? pl * plane : 0) + at;
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(b), 0, 0x7FFFFFFF, 0x00020000);
            uint32_t o = off[u];
            if (tail) o = k0 + kpos[u] < K ? o : kOutside;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(lds + pl * kPlaneBytes + in_plane * 1024u), 16, o, 0, 0, 0);
        }
    }
    // operand of sixteen tile rows from `row16` on (a multiple of 16), k block kk of 32
    static __device__ __forceinline__ s16x8 fragment(const char* lds, int pl, uint32_t row16, int kk, uint32_t lane) {
        const uint32_t g = lane >> 4, i = lane & 15u;
        if constexpr (KC) {
            const uint32_t c = (uint32_t)kk * 4u + g;
            return *reinterpret_cast<const s16x8*>(lds + pl * kPlaneBytes + (row16 + i) * (KT * 2u) + unit_at(i, c) * 16u);
        } else {
            const uint32_t k = 8u * g + (i >> 2);            // (kk * 32 and + 4 leave the swizzle as it is)
            const uint32_t at = (k * TR * 2u + strided_swizzle(k) * 32u + (i & 3u) * 8u) ^ (row16 * 2u);
            const char* p = lds + pl * kPlaneBytes + kk * 32 * TR * 2 + at;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * TR * 2));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// every load of this wave has landed, every LDS read of it is done, and so for the whole workgroup
__device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A workgroup's K loop over one pair of operands: acc[mi][ni] += A rows x B rows.  Wave (wm, wn) of WM x WN owns 16 MI x 16 NI of the tile.
// Two LDS stages: the loads of a step run under the products of the step before.
template <class T, int NP, int KT, int TM, int TN, int WM, int WN, bool AKC, bool BKC, bool PAIR> struct Product {
    static constexpr int WAVES = WM * WN, MI = TM / WM / 16, NI = TN / WN / 16;
    using LA = TileLoad<TM, KT, NP, AKC, WAVES>;
    using LB = TileLoad<TN, KT, NP, BKC, WAVES, PAIR>;
    static constexpr int kStage = LA::kBytes + LB::kBytes;

    template <int ACC> static __device__ __forceinline__ void compute(const char* lds, uint32_t wm, uint32_t wn, uint32_t lane, f32x4 (&acc)[MI][ACC], int at) {
#pragma unroll
        for (int kk = 0; kk < KT / 32; ++kk) {
            s16x8 fa[NP][MI], fb[NP][NI];
#pragma unroll
            for (int p = 0; p < NP; ++p) {
#pragma unroll
                for (int ni = 0; ni < NI; ++ni) fb[p][ni] = LB::fragment(lds + LA::kBytes, p, (wn * NI + ni) * 16u, kk, lane);
#pragma unroll
                for (int mi = 0; mi < MI; ++mi) fa[p][mi] = LA::fragment(lds, p, (wm * MI + mi) * 16u, kk, lane);
            }
#pragma unroll
            for (int pa = 0; pa < NP; ++pa)
#pragma unroll
                for (int pb = 0; pb < NP; ++pb) {
                    if (pa + pb > 2) continue;
#pragma unroll
                    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                        for (int ni = 0; ni < NI; ++ni) acc[mi][at + ni] = mfma16<T>(fb[pb][ni], fa[pa][mi], acc[mi][at + ni]);
                }
        }
    }
    // [k_from, k_to) of the reduction; acc's columns at .. at + NI - 1.  lds0 / lds1: the two stages.  Leaves with every LDS read done.
    template <int ACC> static __device__ __forceinline__ void run(const Operand& A, const Operand& B, const Operand& B2, uint32_t row0, uint32_t col0, uint32_t k_from, uint32_t k_to, char* lds0, char* lds1,
                                                                  f32x4 (&acc)[MI][ACC], int at) {
        const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
        LA la;
        LB lb;
        la.init(A, A, row0, wave, lane);
        lb.init(B, B2, col0, wave, lane);
        auto issue = [&](char* lds, uint32_t k0) {
            la.issue(lds, k0, k_to, wave);
            lb.issue(lds + LA::kBytes, k0, k_to, wave);
        };
        if (k_from < k_to) issue(lds0, k_from);
        for (uint32_t k0 = k_from; k0 < k_to; k0 += 2 * KT) {
            tile_barrier();
            if (k0 + KT < k_to) issue(lds1, k0 + KT);
            compute(lds0, wm, wn, lane, acc, at);
            if (k0 + KT >= k_to) break;
            tile_barrier();
            if (k0 + 2 * KT < k_to) issue(lds0, k0 + 2 * KT);
            compute(lds1, wm, wn, lane, acc, at);
        }
        tile_barrier();
    }
};

// an fp32 number as its three bf16 terms (exact: 8 + 8 + 8 bits); the first is truncated where rounding it would overflow
__device__ __forceinline__ void split3(float v, __bf16 (&t)[3]) {
    t[0] = (__bf16)v;
    if (__builtin_isinf((float)t[0])) t[0] = __builtin_bit_cast(__bf16, (uint16_t)(__builtin_bit_cast(uint32_t, v) >> 16));
    const float r = v - (float)t[0];
    t[1] = (__bf16)r;
    t[2] = (__bf16)(r - (float)t[1]);
}

// four adjacent results as operand planes (T terms): p 8-byte aligned
template <class T, int NP> __device__ __forceinline__ void store_planes(uint16_t* p, uint64_t plane, const float (&v)[4]) {
    if constexpr (NP == 1) {
        Pack<T, 4> o;
#pragma unroll
        for (int r = 0; r < 4; ++r) o.v[r] = from_f32<T>(v[r]);
        *reinterpret_cast<s16x4*>(p) = __builtin_bit_cast(s16x4, o);
    } else {
        Pack<__bf16, 4> o[3];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            __bf16 t[3];
            split3(v[r], t);
#pragma unroll
            for (int q = 0; q < 3; ++q) o[q].v[r] = t[q];
        }
#pragma unroll
        for (int q = 0; q < 3; ++q) *reinterpret_cast<s16x4*>(p + q * plane) = __builtin_bit_cast(s16x4, o[q]);
    }
}

// up to four adjacent results of a row of an output of any alignment: `left` columns of it remain
template <class E> __device__ __forceinline__ void store_row4(E* p, int64_t left, const float (&v)[4]) {
    if (left >= 4) {
        Pack<E, 4> o;
#pragma unroll
        for (int r = 0; r < 4; ++r) o.v[r] = from_f32<E>(v[r]);
        store_pack(p, o);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r < left) p[r] = from_f32<E>(v[r]);
    }
}

}  // namespace envidr
