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

// (an LDS pointer is 32 bits on the device; the compiler's host pass warns about its own 64)
#pragma clang diagnostic ignored "-Wint-to-pointer-cast"

namespace envidr {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) s16x8 lds_s16x8;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4;

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

// a buffer of `bytes` at p; past them a load delivers zeros
__device__ __forceinline__ u32x4 buffer_of(const void* p, uint32_t bytes) {
    const uint64_t b = reinterpret_cast<uint64_t>(p);
    return {(uint32_t)b, (uint32_t)(b >> 32) & 0xFFFFu, bytes, 0x00020000u};
}

// 16 bytes a lane from r + offset to LDS at `lds` + 16 lane.  In assembly because the compiler, which cannot tell the stages apart, would wait
// for every load before the next LDS read: tile_barrier below is the only wait.
__device__ __forceinline__ void load_to_lds(u32x4 r, uint32_t offset, uint32_t lds) {
    uint32_t m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, 0 offen lds\n\ts_mov_b32 m0, %0" : "=&s"(m0) : "s"(lds), "v"(offset), "s"(r) : "memory");
}

// One operand's tile: TR rows x KT k, NP planes.  PAIR: the tile's rows alternate in blocks of 16 between two K-contiguous operands of
// the same shape, each with its own pitch (gate and up weights of the same hidden units land in the same wave).
// The wave loads of a plane (64 x 16 bytes each) go round the waves, so that a wave's loads are a fixed number of LDS rows apart: one offset
// register serves them all, the rest is scalar.  Rows past the operand's end are past the buffer's.
template <int TR, int KT, int NP, bool KC, int WAVES, bool PAIR = false> struct TileLoad {
    static constexpr int kPlaneBytes = TR * KT * 2;
    static constexpr int kBytes = kPlaneBytes * NP;
    static constexpr int kPerPlane = kPlaneBytes / 1024;
    static constexpr int U = (kPerPlane + WAVES - 1) / WAVES;
    static constexpr int kUnits = KC ? KT / 8 : TR / 8;                  // 16-byte units of an LDS row
    static constexpr int kRowsApart = WAVES * 64 / kUnits;               // LDS rows between a wave's loads
    static constexpr int kApart = PAIR ? kRowsApart / 2 : kRowsApart;    // operand rows (K-strided: k) between them
    static_assert(kPlaneBytes % 1024 == 0 && (!PAIR || (KC && kRowsApart % 32 == 0)), "whole wave loads, a wave's of one operand");
    static_assert(U == 1 || kRowsApart % 16 == 0, "one swizzle for a wave's loads");

    const uint16_t* base;
    uint64_t plane;
    uint32_t ld, rows;      // rows of the operand from the tile's first on (K-contiguous)
    uint32_t off, k_of;     // byte offset of the lane's unit from the k-step's base; its first k (K-contiguous)

    // the unit that a row holds at place s, as (row & its swizzle) -- its own inverse
    static __device__ __forceinline__ uint32_t unit_at(uint32_t row, uint32_t s) {
        if constexpr (KC) return s ^ contiguous_swizzle(row);
        else return s ^ (2u * strided_swizzle(row));
    }
    // A 16-byte read takes its 64 lanes in four passes; the first takes lanes 0-3, 12-15 and 20-27, i.e. eight rows of one unit and the other
    // eight of the unit beside it, the second the rest of that half.  With p = the row in 256-byte periods, units p or p ^ 1 (where p's lanes
    // read the other unit) are all different.  (The order 0-15, 16-31, ... would want plain p: measured, that costs every read twice its time.)
    static __device__ __forceinline__ uint32_t contiguous_swizzle(uint32_t row) {
        const uint32_t p = (row / (16u / kUnits)) & (kUnits - 1u);
        return p ^ (KT == 32 ? (p ^ (p >> 1)) & 1u : ((p >> 1) ^ (p >> 2)) & 1u);
    }
    static __device__ __forceinline__ uint32_t strided_swizzle(uint32_t k) {
        if constexpr (TR >= 128) return (k & 3u) | ((k >> 1) & 4u);
        else if constexpr (TR == 64) return ((k >> 1) & 1u) | ((k >> 2) & 2u);
        else return (k >> 3) & 1u;
    }

    __device__ __forceinline__ void init(const Operand& a, const Operand& a2, uint32_t row0, uint32_t wave, uint32_t lane) {
        const uint32_t idx = wave * 64u + lane, r = idx / kUnits, c = unit_at(r, idx % kUnits);
        const bool second = PAIR && (wave * 64u / kUnits >> 4 & 1u);
        plane = second ? a2.plane : a.plane;
        ld = second ? a2.ld : a.ld;
        base = (second ? a2.p : a.p) + (KC ? (uint64_t)row0 * ld : (uint64_t)row0);
        if constexpr (KC) {
            off = ((PAIR ? (r >> 5) * 16u + (r & 15u) : r) * ld + c * 8u) * 2u;
            k_of = c * 8u;
            rows = row0 < a.ext ? min(a.ext - row0, (uint32_t)TR) : 0u;
        } else {
            off = row0 + c * 8u < a.ext ? (r * ld + c * 8u) * 2u : kOutside;
        }
    }
    // starts the loads of the step that begins at k0 (of K) into `lds`
    __device__ __forceinline__ void issue(uint32_t lds, uint32_t k0, uint32_t K, uint32_t wave) const {
        const uint16_t* b = base + (KC ? (uint64_t)k0 : (uint64_t)k0 * ld);
        const uint32_t left = KC ? rows : (k0 < K ? min(K - k0, (uint32_t)KT) : 0u);
        uint32_t o = off;
        if constexpr (KC) o = k0 + k_of < K ? o : kOutside;
#pragma unroll
        for (int pl = 0; pl < NP; ++pl) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (kPerPlane % WAVES != 0 && u * WAVES + wave >= (uint32_t)kPerPlane) break;
                const uint32_t here = left > (uint32_t)(u * kApart) ? (left - u * kApart) * ld * 2u : 0u;
                load_to_lds(buffer_of(b + pl * plane + (uint64_t)(u * kApart) * ld, here), o, lds + pl * kPlaneBytes + (u * WAVES + wave) * 1024u);
            }
        }
    }
    // operand of sixteen tile rows from `row16` on (a multiple of 16), k block kk of 32; lds: the tile's LDS address.  (The K-strided form adds
    // the tile's address before the exclusive or: that way the addresses of a step are formed in the step and take no registers across it.)
    static __device__ __forceinline__ s16x8 fragment(uint32_t lds, int pl, uint32_t row16, int kk, uint32_t lane) {
        const uint32_t g = lane >> 4, i = lane & 15u;
        if constexpr (KC) {
            const uint32_t at = lds + i * (KT * 2u) + unit_at(i, (uint32_t)kk * 4u + g) * 16u;
            return *(const lds_s16x8*)(at + pl * kPlaneBytes + row16 * (KT * 2u));
        } else {
            const uint32_t k = 8u * g + (i >> 2);            // (kk * 32 and + 4 leave the swizzle as it is)
            const uint32_t at = (lds + k * TR * 2u + strided_swizzle(k) * 32u + (i & 3u) * 8u) ^ (row16 * 2u & 255u);
            const uint32_t p = at + (row16 * 2u & ~255u) + pl * kPlaneBytes + kk * 32 * TR * 2;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * TR * 2));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// At most N of this wave's LDS-direct loads are still in flight, every LDS read of it is done, and so for the whole workgroup
template <int N> __device__ __forceinline__ void tile_barrier() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }

// Every LDS operation of the workgroup is done.  (__syncthreads would wait for memory too)
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A workgroup's K loop over one pair of operands: acc[mi][ni] += A rows x B rows.  Wave (wm, wn) of WM x WN owns 16 MI x 16 NI of the tile.
// Memory -> LDS: S stages of KT, S steps ahead; LDS -> registers: 32 k ahead, so that the reads run under the products of the 32 before
// (the waves of a workgroup pass the barrier together: without this they would all read, then all multiply).
//   barrier t: step t + 1 has landed for everyone, and everyone has the last of step t in registers, so its stage is free for step t + S
// Steps past the end are loads of zeros: the number in flight is the same at every wait.
// (B's tile may be loaded TL wide and used TN wide: a K-strided tile's rows have to divide a bank period.)
template <class T, int NP, int TM, int TN, int WM, int WN, bool AKC, bool BKC, bool PAIR, int TL = TN> struct Product {
    static constexpr int KT = NP == 1 ? 64 : 32;
    static constexpr int WAVES = WM * WN, MI = TM / WM / 16, NI = TN / WN / 16;
    using LA = TileLoad<TM, KT, NP, AKC, WAVES>;
    using LB = TileLoad<TL, KT, NP, BKC, WAVES, PAIR>;
    static constexpr int kStage = LA::kBytes + LB::kBytes;

    struct Fragments {
        s16x8 a[NP][MI], b[NP][NI];
    };
    static __device__ __forceinline__ void read_a(uint32_t lds, int kk, int p, uint32_t wm, uint32_t lane, s16x8 (&a)[MI]) {
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) a[mi] = LA::fragment(lds, p, (wm * MI + mi) * 16u, kk, lane);
    }
    static __device__ __forceinline__ void read_b(uint32_t lds, int kk, int p, uint32_t wn, uint32_t lane, s16x8 (&b)[NI]) {
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) b[ni] = LB::fragment(lds + LA::kBytes, p, (wn * NI + ni) * 16u, kk, lane);
    }
    static __device__ __forceinline__ void read(uint32_t lds, int kk, uint32_t wm, uint32_t wn, uint32_t lane, Fragments& f) {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            read_b(lds, kk, p, wn, lane, f.b[p]);
            read_a(lds, kk, p, wm, lane, f.a[p]);
        }
    }
    template <int ACC> static __device__ __forceinline__ void multiply(const s16x8 (&a)[MI], const s16x8 (&b)[NI], f32x4 (&acc)[MI][ACC], int at) {
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) acc[mi][at + ni] = mfma16<T>(b[ni], a[mi], acc[mi][at + ni]);
    }
    // the products of the step in `f`; `next`: the step behind it, read from `lds`
    template <int ACC> static __device__ __forceinline__ void step(uint32_t lds, int kk, uint32_t wm, uint32_t wn, uint32_t lane, Fragments& f, Fragments& next, f32x4 (&acc)[MI][ACC], int at) {
        if constexpr (NP == 1) {
            read(lds, kk, wm, wn, lane, next);
            multiply(f.a[0], f.b[0], acc, at);
        } else {
            // the small products first; a term's registers take the next step's as soon as its last product is out
            multiply(f.a[0], f.b[2], acc, at);
            read_b(lds, kk, 2, wn, lane, next.b[2]);
            multiply(f.a[2], f.b[0], acc, at);
            read_a(lds, kk, 2, wm, lane, next.a[2]);
            multiply(f.a[1], f.b[1], acc, at);
            multiply(f.a[0], f.b[1], acc, at);
            read_b(lds, kk, 1, wn, lane, next.b[1]);
            multiply(f.a[1], f.b[0], acc, at);
            read_a(lds, kk, 1, wm, lane, next.a[1]);
            read_a(lds, kk, 0, wm, lane, next.a[0]);
            read_b(lds, kk, 0, wn, lane, next.b[0]);
            multiply(f.a[0], f.b[0], acc, at);
        }
    }
    // The loads' side of the pipeline: where the next step comes from.
    struct Source {
        LA la;
        LB lb;
        uint32_t ahead, to;
        __device__ __forceinline__ void init(const Operand& A, const Operand& B, const Operand& B2, uint32_t row0, uint32_t col0, uint32_t k_from, uint32_t k_to) {
            const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
            la.init(A, A, row0, wave, lane);
            lb.init(B, B2, col0, wave, lane);
            ahead = k_from;
            to = k_to;
        }
        __device__ __forceinline__ void issue(uint32_t lds) {
            const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
            la.issue(lds, ahead, to, wave);
            lb.issue(lds + LA::kBytes, ahead, to, wave);
            ahead += KT;
        }
    };
    // steps of a reduction of length k: at least the two that are under way before it starts, an even number where the registers' roles alternate
    static __device__ __forceinline__ uint32_t steps(uint32_t k) {
        const uint32_t n = (k + KT - 1) / KT;
        return KT == 32 ? (n < 2 ? 2u : (n + 1u) & ~1u) : (n < 2 ? 2u : n);
    }
    // acc's columns at .. at + NI - 1 += the n steps whose first two are under way into the stages `stage`, stage_bytes - `stage` (offsets from
    // lds) from `src`.  `turn` is called when all loads of these steps are out; issue_next(lds) then starts the steps of what comes next: two of
    // them are under way on return, the first into `stage`.
    // relaxed: exactly STORES memory operations were issued behind the first two steps' loads (the tile before's results); they may stay
    // in flight while those steps are waited for -- operations complete in order, so "all but the last STORES" are the loads.
    template <int STORES, int ACC, class Turn, class Issue>
    static __device__ __forceinline__ void run(uint32_t lds, uint32_t stage_bytes, uint32_t& stage, Source& src, uint32_t n, bool relaxed, f32x4 (&acc)[MI][ACC], int at, Turn turn, Issue issue_next) {
        static_assert(STORES < 64, "the counter of operations in flight holds 63");
        const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
        Fragments f[2];
        auto barrier = [&](bool first) {
            if (STORES > 0 && first && relaxed) tile_barrier<STORES>();
            else tile_barrier<0>();
        };
        barrier(true);
        read(lds + stage, 0, wm, wn, lane, f[0]);
        auto one = [&](Fragments& now, Fragments& then, bool first, bool last) {
            const uint32_t other = stage_bytes - stage;
            if constexpr (KT == 64) step(lds + stage, 1, wm, wn, lane, now, then, acc, at);
            barrier(first);
            if (!last) src.issue(lds + stage); else issue_next(lds + stage);
            if constexpr (KT == 64) step(lds + other, 0, wm, wn, lane, then, now, acc, at);
            else step(lds + other, 0, wm, wn, lane, now, then, acc, at);
            stage = other;
        };
        if constexpr (KT == 64) {
            for (uint32_t s = 0; s + 2 < n; ++s) one(f[0], f[1], s == 0, false);
            turn();
            one(f[0], f[1], n == 2, true);
            one(f[0], f[1], false, true);
        } else {
            for (uint32_t s = 0; s + 2 < n; s += 2) {
                one(f[0], f[1], s == 0, false);
                one(f[1], f[0], false, false);
            }
            turn();
            one(f[0], f[1], n == 2, true);
            one(f[1], f[0], false, true);
        }
    }
};

// A workgroup's share of the tiles.  Workgroups go to the eight XCDs in turn: each XCD gets a run of adjacent tiles, column tiles first, so that
// the rows of a run and the weights stay in its own L2; its workgroups walk the run side by side.
struct TileWalk {
    uint32_t now, end, by;
    __device__ __forceinline__ TileWalk(uint32_t tiles) {
        const uint32_t each = (tiles + 7u) / 8u, first = (blockIdx.x & 7u) * each;
        now = first + (blockIdx.x >> 3);
        end = min(first + each, tiles);
        by = gridDim.x >> 3;
    }
    __device__ __forceinline__ bool valid() const { return now < end; }
    __device__ __forceinline__ bool more() const { return now + by < end; }
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

// one memory operation, dropped by the lanes whose offset is past the `bytes` at p
__device__ __forceinline__ void store_to_buffer(u32x4 v, void* p, uint32_t bytes, uint32_t offset) {
    __builtin_amdgcn_raw_buffer_store_b128(v, __builtin_amdgcn_make_buffer_rsrc(p, 0, bytes, 0x00020000), offset, 0, 0);
}

// Sixteen-bit results on their way out.  A wave holds, of each row of a 16-row block, four adjacent columns in each lane group: stored like
// that a row is written 32 bytes at a time.  Through 2 KiB of LDS of its own the wave turns kRows rows of COLS columns into whole rows.
template <int COLS> struct RowStore {
    static constexpr int kPitch = COLS <= 16 ? 16 : COLS <= 32 ? 32 : 64;           // of a row in LDS
    static constexpr int kRows = 1024 / kPitch, kUnits = kPitch / 8, kStores = 2;
    static_assert(COLS % 16 == 0 && COLS <= 64, "whole blocks");
    typedef __attribute__((address_space(3))) s16x4 lds_half;
    // columns col .. col + 3 of row `row` of the block
    static __device__ __forceinline__ void put(uint32_t lds, uint32_t row, uint32_t col, s16x4 v) {
        const uint32_t unit = (col >> 3) ^ (row & (kUnits - 1u));
        *(lds_half*)(lds + row * (kPitch * 2u) + unit * 16u + (col & 4u) * 2u) = v;
    }
    static __device__ __forceinline__ u32x4 unit_of(uint32_t lds, uint32_t row, uint32_t unit) { return *(const lds_u32x4*)(lds + row * (kPitch * 2u) + (unit ^ (row & (kUnits - 1u))) * 16u); }
    // the block's rows to p (its first row, `rows` of them there) from column col0 on (`cols` of them there): 16-byte aligned, whole units.
    // Always kStores memory operations.
    static __device__ __forceinline__ void flush(uint32_t lds, uint16_t* p, uint32_t ld, uint32_t rows, uint32_t col0, uint32_t cols) {
        const uint32_t lane = threadIdx.x & 63u;
        const uint32_t bytes = min(rows, (uint32_t)kRows) * ld * 2u;
#pragma unroll
        for (int j = 0; j < kStores; ++j) {
            const uint32_t idx = j * 64u + lane, row = idx / kUnits, unit = idx % kUnits, col = col0 + unit * 8u;
            store_to_buffer(unit_of(lds, row, unit), p, bytes, unit * 8u < (uint32_t)COLS && col < cols ? (row * ld + col) * 2u : kOutside);
        }
    }
    // the same to an output of any alignment and width (148664 x 899 of bf16: 142 us; stored four columns a lane, 32 bytes of a row at a time, 257)
    static __device__ __forceinline__ void flush_any(uint32_t lds, uint16_t* p, int64_t ld, uint32_t rows, uint32_t col0, uint32_t cols) {
        const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
        for (int j = 0; j < kStores; ++j) {
            const uint32_t idx = j * 64u + lane, row = idx / kUnits, unit = idx % kUnits, col = col0 + unit * 8u;
            const Pack<uint16_t, 8> v = __builtin_bit_cast(Pack<uint16_t, 8>, unit_of(lds, row, unit));
            if (row >= rows || unit * 8u >= (uint32_t)COLS || col >= cols) continue;
            uint16_t* to = p + (int64_t)row * ld + col;
            if (cols - col >= 8u) {
                store_pack(to, v);
            } else {
#pragma unroll
                for (int r = 0; r < 7; ++r)
                    if (col + r < cols) to[r] = v.v[r];
            }
        }
    }
};

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

template <class T> __device__ __forceinline__ s16x4 pack4(const float (&v)[4]) {
    Pack<T, 4> o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o.v[r] = from_f32<T>(v[r]);
    return __builtin_bit_cast(s16x4, o);
}

// A wave's results acc[MI][NI], its rows from row0 and columns from col0 on, to out [rows][cols] with pitch ld.  aligned: whole 16-byte units
// everywhere, and then exactly kCount memory operations.  scratch: 2 KiB of LDS (16-bit results).
template <class E, int MI, int NI> struct ResultStore {
    static constexpr bool kWide = sizeof(E) == 4;
    static constexpr int kCount = kWide ? MI * NI : MI * 16 / RowStore<NI * 16>::kRows * 2;
    static __device__ __forceinline__ void store(uint32_t scratch, const f32x4 (&acc)[MI][NI], E* out, int64_t ld, uint32_t rows, uint32_t cols, uint32_t row0, uint32_t col0, bool aligned) {
        const uint32_t lane = threadIdx.x & 63u, i = lane & 15u, g = lane >> 4;
        if constexpr (kWide) {
            if (!aligned) {
#pragma unroll
                for (int mi = 0; mi < MI; ++mi) {
                    const uint32_t m = row0 + mi * 16u + i;
                    if (m >= rows) continue;
#pragma unroll
                    for (int ni = 0; ni < NI; ++ni) {
                        const uint32_t n = col0 + ni * 16u + 4u * g;
                        const float v[4] = {acc[mi][ni][0], acc[mi][ni][1], acc[mi][ni][2], acc[mi][ni][3]};
                        store_row4(out + (int64_t)m * ld + n, (int64_t)cols - n, v);
                    }
                }
                return;
            }
#pragma unroll
            for (int mi = 0; mi < MI; ++mi) {
                const uint32_t m0 = row0 + mi * 16u, left = m0 < rows ? min(rows - m0, 16u) : 0u;
#pragma unroll
                for (int ni = 0; ni < NI; ++ni) {
                    const uint32_t n = col0 + ni * 16u + 4u * g;
                    store_to_buffer(__builtin_bit_cast(u32x4, acc[mi][ni]), out + (int64_t)m0 * ld, left * (uint32_t)ld * 4u, n < cols ? (i * (uint32_t)ld + n) * 4u : kOutside);
                }
            }
        } else {
            using W = RowStore<NI * 16>;
#pragma unroll
            for (int mi = 0; mi < MI; ++mi) {
#pragma unroll
                for (int ni = 0; ni < NI; ++ni) {
                    const float v[4] = {acc[mi][ni][0], acc[mi][ni][1], acc[mi][ni][2], acc[mi][ni][3]};
                    W::put(scratch, mi * 16u % W::kRows + i, ni * 16u + 4u * g, pack4<E>(v));
                }
                if ((mi + 1) * 16 % W::kRows == 0) {
                    const uint32_t m0 = row0 + (mi + 1) * 16u - W::kRows, left = m0 < rows ? rows - m0 : 0u;
                    uint16_t* p = reinterpret_cast<uint16_t*>(out + (int64_t)m0 * ld);
                    if (aligned) W::flush(scratch, p, (uint32_t)ld, left, col0, cols);
                    else W::flush_any(scratch, p, ld, left, col0, cols);
                }
            }
        }
    }
};

// Rows of 32-bit values on their way to an operand of the next product: COLS columns of kRows rows, as NP planes
template <class T, int NP, int COLS> struct PlaneStore {
    using W = RowStore<COLS>;
    static constexpr int kBlocks = W::kRows / 16, kCount = 2 * NP;       // 16-row blocks, memory operations
    // v[block][nj][r]: column 16 nj + 4 (lane / 16) + r of row 16 block + lane % 16
    static __device__ __forceinline__ void store(uint32_t scratch, const float (&v)[kBlocks][COLS / 16][4], uint16_t* out, uint64_t plane, uint32_t ld, uint32_t rows, uint32_t row0, uint32_t col0, uint32_t cols) {
        const uint32_t lane = threadIdx.x & 63u;
        float rest[kBlocks][COLS / 16][4];
#pragma unroll
        for (int p = 0; p < NP; ++p) {
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int j = 0; j < COLS / 16; ++j) {
                    s16x4 o;
                    if constexpr (NP == 1) {
                        o = pack4<T>(v[b][j]);
                    } else {
                        // (the terms one after the other, as split3 makes them)
                        Pack<__bf16, 4> t;
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float x = p == 0 ? v[b][j][r] : rest[b][j][r];
                            t.v[r] = (__bf16)x;
                            if (p == 0 && __builtin_isinf((float)t.v[r])) t.v[r] = __builtin_bit_cast(__bf16, (uint16_t)(__builtin_bit_cast(uint32_t, x) >> 16));
                            rest[b][j][r] = x - (float)t.v[r];
                        }
                        o = __builtin_bit_cast(s16x4, t);
                    }
                    W::put(scratch, b * 16u + (lane & 15u), j * 16u + 4u * (lane >> 4), o);
                }
            W::flush(scratch, out + p * plane + (uint64_t)row0 * ld, ld, row0 < rows ? rows - row0 : 0u, col0, cols);
        }
    }
};

// Eight adjacent elements from column k of a row of n; zeros behind it.  whole: n is a multiple of 8, and a load behind it is a load of the last
// eight instead, made zero: no branch, so that loads can go out together.
template <class E> __device__ __forceinline__ s16x8 load8(const E* row, uint32_t k, uint32_t n, bool whole) {
    if (whole) {
        const s16x8 v = __builtin_bit_cast(s16x8, load_pack<E, 8>(row + min(k, n - 8u)));
        return k < n ? v : s16x8{};
    }
    if (k + 8u <= n) return __builtin_bit_cast(s16x8, load_pack<E, 8>(row + k));
    Pack<E, 8> v;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) v.v[i] = k + i < n ? row[k + i] : from_f32<E>(0.0f);
    return __builtin_bit_cast(s16x8, v);
}

}  // namespace envidr
