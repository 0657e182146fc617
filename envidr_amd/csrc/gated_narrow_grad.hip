// The gated feed-forward block of narrow layers, backward (16-bit types): dx, dWg, dWu and dWd in one pass over the rows, nothing of the hidden
// layer through memory.
//
// A workgroup's eight waves form teams of `slices` waves; a team takes 32 rows at a time, a wave 32 hidden units of them.  The gate and up matrices
// lie in LDS (in registers the sums of their gradients leave no room for them).  Per 32 rows:
//   1. g, u, dh (x and dy from LDS) -> h, dg, du, rounded to the type, into LDS as [row][unit]; a lane's eight units {4 q .. 4 q + 3, 16 + 4 q ..
//      16 + 4 q + 3} (q = lane / 16) are one 16-byte unit there, so units lie in that order;
//   2. dWg += dg^T x, dWu += du^T x, dWd += dy^T h: the reduction over the rows is one k step of the matrix core; both operands are transposing
//      reads, of columns that the wave wrote itself, the sums stay in registers from the first row to the last;
//   3. behind a barrier, since a team's waves need each other's units: dx = dg Wg + du Wu, a block of 16 columns a wave, the weights from LDS; the
//      results go through x's place in LDS, so that rows are written whole (10^6 rows of 32 -> 64 -> 12: 127 us; in blocks of 16 columns 145).
// Next rows are loaded under the present ones' work and follow dx there.  At the end the teams' sums are added up in LDS and the
// workgroup's go to `part`; k_sum_splits adds those of all workgroups, in order.
// LDS rows are an odd multiple of 32 bytes apart: sixteen-byte reads of sixteen rows and transposing reads of eight rows both find them on
// different banks (for the transposing ones the rows of a k step are taken as 4 q .. 4 q + 3, 16 + 4 q .. 16 + 4 q + 3).
// Bound: the phases' latencies with two waves a SIMD (the sums take half the registers): vector ALU 35 %, LDS 26 %, matrix cores 20 % busy.
// 146 000 rows of 72 -> 256 -> 12 in bf16: 93 us and 8 for the parts; through memory (hidden layer's operands, products, transposed products) 198.
#include "gated_mlp.hip.h"
#include "gemm_core.hip.h"

#include <type_traits>

namespace envidr {
namespace {

constexpr int kLds = 160 * 1024, kWaves = kTeamWaves, kTeamRows = 32;
constexpr uint32_t kDyPitch = 96;

// an operand of sixteen columns and 32 rows (k) from `at`: rows 4 q .. and 16 + 4 q .. of the lane groups q
__device__ __forceinline__ s16x8 columns(uint32_t at, uint32_t pitch, uint32_t lane) {
    const uint32_t p = at + (lane >> 2) * pitch + (lane & 3u) * 8u;              // (4 (lane / 16) + lane % 16 / 4 = lane / 4)
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 16u * pitch));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Units behind the last one have weights of zero, which an infinity in x or dy makes NaN, and dx takes all units of a team: they are cleared.  All ones
// for those of a lane's eight units that are there.  (From a lane number that the compiler takes for a new one: what it kept of this across the
// loop over the rows would be spilled.)
__device__ __forceinline__ s16x8 present_units(uint32_t lane, uint32_t first, uint32_t F) {
    asm volatile("" : "+v"(lane));
    const uint32_t f = first + 4u * (lane >> 4);
    s16x8 keep;
#pragma unroll
    for (uint32_t n = 0; n < 8; ++n) keep[n] = f + 16u * (n >> 2) + (n & 3u) < F ? -1 : 0;
    return keep;
}

// DB: blocks of 16 input columns; ONE: one team, whose rows are one 16-byte unit a thread at most
template <class E, int ACT, int DB, bool ONE> __global__ void __launch_bounds__(kWaves * 64, 2) k_narrow_backward(NarrowGradArgs a) {
    constexpr int KD = (DB + 1) / 2;                                             // k blocks of 32 of them
    constexpr uint32_t kXPitch = KD * 64 + 32;
    constexpr int kXUnits = ONE ? 1 : 2 * KD, kDyUnits = ONE ? 1 : 2;            // 16-byte units a thread carries, at most
    __shared__ __attribute__((aligned(1024))) char lds_all[kLds];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, i = lane & 15u;
    const uint32_t slices = ONE ? kWaves : a.slices, team = ONE ? 0u : wave / slices, slice = ONE ? wave : wave % slices, teams = kWaves / slices, blocks = (a.D + 15u) / 16u;
    const uint32_t used = ONE ? (a.F + 63u) / 64u * 2u : (a.F + 31u) / 32u;         // blocks of 32 units that dx is formed of (ONE: in pairs)
    const uint32_t h_pitch = slices * 64u + 32u, hidden = slices * 32u;
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_void*)lds_all, lds_w = lds, team_bytes = kTeamRows * (kXPitch + kDyPitch + 2u * h_pitch), teams_at = lds + 2u * hidden * kXPitch;
    const uint32_t xs = teams_at + team * team_bytes, ys = xs + kTeamRows * kXPitch, dgs = ys + kTeamRows * kDyPitch, dus = dgs + kTeamRows * h_pitch;
    const E *wg = static_cast<const E*>(a.wg), *wu = static_cast<const E*>(a.wu), *wd = static_cast<const E*>(a.wd);
    const bool whole_x = a.D % 8u == 0u, whole_y = a.O % 8u == 0u;
    const uint32_t rows = teams * kTeamRows, tiles = (a.M + rows - 1u) / rows;

    auto x_unit = [&](uint32_t n) { return teams_at + n / (KD * 4u) / kTeamRows * team_bytes + n / (KD * 4u) % kTeamRows * kXPitch + n % (KD * 4u) * 16u; };
    // the next rows of x and dy, and where they go: unit n of a tile is row n / units, zeros behind the last row and column
    s16x8 nx[kXUnits], ny[kDyUnits];
    auto fetch = [&](uint32_t t) {
#pragma unroll
        for (int j = 0; j < kXUnits; ++j) {
            const uint32_t n = j * (kWaves * 64u) + threadIdx.x, r = n / (KD * 4u), m = t * rows + r;
            if (r < rows) nx[j] = m < a.M ? load8(static_cast<const E*>(a.x) + (int64_t)m * a.ldx, n % (KD * 4u) * 8u, a.D, whole_x) : s16x8{};
        }
#pragma unroll
        for (int j = 0; j < kDyUnits; ++j) {
            const uint32_t n = j * (kWaves * 64u) + threadIdx.x, r = n / 4u, m = t * rows + r;
            if (r < rows) ny[j] = m < a.M ? load8(static_cast<const E*>(a.dy) + (int64_t)m * a.lddy, n % 4u * 8u, a.O, whole_y) : s16x8{};
        }
    };
    auto put = [&] {
#pragma unroll
        for (int j = 0; j < kXUnits; ++j) {
            const uint32_t n = j * (kWaves * 64u) + threadIdx.x, r = n / (KD * 4u);
            if (r < rows) *(lds_s16x8*)(x_unit(n)) = nx[j];
        }
#pragma unroll
        for (int j = 0; j < kDyUnits; ++j) {
            const uint32_t n = j * (kWaves * 64u) + threadIdx.x, r = n / 4u;
            if (r < rows) *(lds_s16x8*)(teams_at + r / kTeamRows * team_bytes + kTeamRows * kXPitch + r % kTeamRows * kDyPitch + n % 4u * 16u) = ny[j];
        }
    };
    // dx of tile t, which has taken x's place in LDS: whole rows, the units that this thread puts the next x into
    auto store_dx = [&](uint32_t t) {
#pragma unroll
        for (int j = 0; j < kXUnits; ++j) {
            const uint32_t n = j * (kWaves * 64u) + threadIdx.x, r = n / (KD * 4u), c = n % (KD * 4u) * 8u, m = t * rows + r;
            if (r >= rows || m >= a.M || c >= a.D) continue;
            const Pack<E, 8> v = __builtin_bit_cast(Pack<E, 8>, *(const lds_s16x8*)(x_unit(n)));
            E* to = static_cast<E*>(a.dx) + (int64_t)m * a.lddx + c;
            if (a.D - c >= 8u) {
                store_pack(to, v);
            } else {
#pragma unroll
                for (uint32_t q = 0; q < 7; ++q)
                    if (c + q < a.D) to[q] = v.v[q];
            }
        }
    };
    uint32_t t = blockIdx.x;                                                     // (the grid has no more workgroups than tiles)
    fetch(t);
    // weights: gate and up in LDS (rows of units), the wave's part of Wd, transposed, in registers
    for (uint32_t n = threadIdx.x; n < 2u * hidden * (KD * 4u); n += kWaves * 64u) {
        const uint32_t row = n / (KD * 4u), unit = n % (KD * 4u), f = row % hidden;
        s16x8 v = {};
        if (f < a.F) v = load8(row < hidden ? wg + (int64_t)f * a.lg : wu + (int64_t)f * a.lu, unit * 8u, a.D, whole_x);
        *(lds_s16x8*)(lds_w + row * kXPitch + unit * 16u) = v;
    }
    s16x8 rd[2];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const uint32_t f = slice * 32u + b * 16u + i;
        Pack<E, 8> v;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) v.v[j] = f < a.F && g * 8u + j < a.O ? wd[(int64_t)(g * 8u + j) * a.ldn + f] : from_f32<E>(0.0f);
        rd[b] = __builtin_bit_cast(s16x8, v);
    }
    f32x4 sum_g[2][DB] = {}, sum_u[2][DB] = {}, sum_d[2][2] = {};
    put();
    __syncthreads();
    for (;;) {
        const bool more = t + gridDim.x < tiles;
        if (more) fetch(t + gridDim.x);
        using Units8 = Pack<E, 8>;
        Units8 vh[2], vg[2], vu[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            f32x4 pg[2] = {}, pu[2] = {}, dh[2];
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) dh[rb] = mfma16<E>(rd[b], *(const lds_s16x8*)(ys + (rb * 16u + i) * kDyPitch + g * 16u), f32x4{});
#pragma unroll
            for (int kk = 0; kk < KD; ++kk) {
                const uint32_t at = lds_w + (slice * 32u + b * 16u + i) * kXPitch + (kk * 4u + g) * 16u;
                const s16x8 w = *(const lds_s16x8*)at, v = *(const lds_s16x8*)(at + hidden * kXPitch);
#pragma unroll
                for (int rb = 0; rb < 2; ++rb) {
                    const s16x8 x = *(const lds_s16x8*)(xs + (rb * 16u + i) * kXPitch + (kk * 4u + g) * 16u);
                    pg[rb] = mfma16<E>(w, x, pg[rb]);
                    pu[rb] = mfma16<E>(v, x, pu[rb]);
                }
            }
#pragma unroll
            for (int rb = 0; rb < 2; ++rb)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float act, slope;
                    activation<ACT, false>(pg[rb][q], act, slope);
                    vh[rb].v[4 * b + q] = from_f32<E>(act * pu[rb][q]);
                    vg[rb].v[4 * b + q] = from_f32<E>(dh[rb][q] * pu[rb][q] * slope);
                    vu[rb].v[4 * b + q] = from_f32<E>(dh[rb][q] * act);
                }
        }
        if constexpr (!ONE) {
            if (slice * 32u + 32u > a.F) {
                const s16x8 keep = present_units(lane, slice * 32u, a.F);
#pragma unroll
                for (int rb = 0; rb < 2; ++rb) {
                    vg[rb] = __builtin_bit_cast(Units8, (s16x8)(__builtin_bit_cast(s16x8, vg[rb]) & keep));
                    vu[rb] = __builtin_bit_cast(Units8, (s16x8)(__builtin_bit_cast(s16x8, vu[rb]) & keep));
                }
            }
        }
        s16x8 du[2];
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
            // (rows behind the last one: zeros, not what weights that are infinite make of zeros)
            const uint32_t row = rb * 16u + i, at = row * h_pitch + (slice * 4u + g) * 16u;
            const bool inside = t * rows + team * kTeamRows + row < a.M;
            *(lds_s16x8*)(dgs + at) = inside ? __builtin_bit_cast(s16x8, vg[rb]) : s16x8{};
            *(lds_s16x8*)(dus + at) = inside ? __builtin_bit_cast(s16x8, vh[rb]) : s16x8{};        // (du's place, until h has been read back)
            du[rb] = inside ? __builtin_bit_cast(s16x8, vu[rb]) : s16x8{};
        }
        // (LDS operations of a wave are done in their order; the compiler has to leave them in it: lanes read what others wrote)
        asm volatile("" ::: "memory");
        s16x8 h[2], ty[2];
        if (a.want_w) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                h[c] = columns(dus + slice * 64u + c * 32u, h_pitch, lane);
                ty[c] = columns(ys + c * 32u, kDyPitch, lane);
            }
        }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) *(lds_s16x8*)(dus + (rb * 16u + i) * h_pitch + (slice * 4u + g) * 16u) = du[rb];
        asm volatile("" ::: "memory");
        if (a.want_w) {
            s16x8 tg[2], tu[2], tx[DB];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                tg[c] = columns(dgs + slice * 64u + c * 32u, h_pitch, lane);
                tu[c] = columns(dus + slice * 64u + c * 32u, h_pitch, lane);
            }
#pragma unroll
            for (int d = 0; d < DB; ++d) tx[d] = columns(xs + d * 32u, kXPitch, lane);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int o = 0; o < 2; ++o) sum_d[c][o] = mfma16<E>(h[c], ty[o], sum_d[c][o]);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    sum_g[c][d] = mfma16<E>(tx[d], tg[c], sum_g[c][d]);
                    sum_u[c][d] = mfma16<E>(tx[d], tu[c], sum_u[c][d]);
                }
            }
        }
        if constexpr (ONE) {                 // (here, where nothing but the sums is in registers, as these are short)
            if (slice * 32u + 32u > a.F && slice < used) {
                const s16x8 keep = present_units(lane, slice * 32u, a.F);
                uint32_t l = lane;
                asm volatile("" : "+v"(l));
                const uint32_t at = (l & 15u) * h_pitch + (slice * 4u + (l >> 4)) * 16u;
#pragma unroll
                for (uint32_t rb = 0; rb < 2; ++rb) {
                    lds_s16x8 *pg = (lds_s16x8*)(dgs + at + rb * 16u * h_pitch), *pu = (lds_s16x8*)(dus + at + rb * 16u * h_pitch);
                    *pg &= keep;
                    *pu &= keep;
                }
            }
        }
        lds_barrier();
        if (a.dx) {
#pragma unroll 1
            for (uint32_t d = slice; d < blocks; d += slices) {
                f32x4 p[2][2] = {};
                // (the next units' reads under the present ones' products)
                struct Units {
                    s16x8 w[2], h[2][2];
                } now, next;
                auto read = [&](Units& u, uint32_t hb) {
                    u.w[0] = columns(lds_w + hb * 32u * kXPitch + d * 32u, kXPitch, lane);
                    u.w[1] = columns(lds_w + (hidden + hb * 32u) * kXPitch + d * 32u, kXPitch, lane);
#pragma unroll
                    for (int rb = 0; rb < 2; ++rb) {
                        const uint32_t at = (rb * 16u + i) * h_pitch + (hb * 4u + g) * 16u;
                        u.h[0][rb] = *(const lds_s16x8*)(dgs + at);
                        u.h[1][rb] = *(const lds_s16x8*)(dus + at);
                    }
                };
                auto multiply = [&](const Units& u) {
#pragma unroll
                    for (int rb = 0; rb < 2; ++rb)
#pragma unroll
                        for (int m = 0; m < 2; ++m) p[m][rb] = mfma16<E>(u.w[m], u.h[m][rb], p[m][rb]);
                };
                if constexpr (ONE) {
                    read(now, 0);
#pragma unroll 1
                    for (uint32_t hb = 0; hb < used; hb += 2) {
                        read(next, hb + 1);
                        multiply(now);
                        if (hb + 2 < used) read(now, hb + 2);
                        multiply(next);
                    }
                } else {                     // (two sets of operands and several teams' rows would not fit the registers)
#pragma unroll 1
                    for (uint32_t hb = 0; hb < used; ++hb) {
                        read(now, hb);
                        multiply(now);
                    }
                }
#pragma unroll
                for (int rb = 0; rb < 2; ++rb) {
                    const f32x4 v = p[0][rb] + p[1][rb];
                    *(lds_s16x4*)(xs + (rb * 16u + i) * kXPitch + d * 32u + g * 8u) = pack4<E>({v[0], v[1], v[2], v[3]});
                }
            }
            lds_barrier();
            store_dx(t);
        }
        if (!more) break;
        put();
        lds_barrier();
        t += gridDim.x;
    }
    if (!a.want_w) return;
    // team 0 adds the others' sums to its own, one team after the other
    constexpr int kSums = 4 * DB + 4;
    auto each = [&](auto f) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                f(sum_g[c][d], (2 * c) * DB + d);
                f(sum_u[c][d], (2 * c + 1) * DB + d);
            }
#pragma unroll
            for (int o = 0; o < 2; ++o) f(sum_d[c][o], 4 * DB + 2 * c + o);
        }
    };
    for (uint32_t other = 1; other < teams; ++other) {
        const uint32_t at = lds + slice * (kSums * 1024u) + lane * 16u;
        __syncthreads();
        if (team == other) each([&](f32x4& s, int n) { *(lds_f32x4*)(at + n * 1024u) = s; });
        __syncthreads();
        if (team == 0) each([&](f32x4& s, int n) { s += *(const lds_f32x4*)(at + n * 1024u); });
    }
    if (team != 0) return;
    // (place p = 8 q + 4 b + r of a slice is unit 16 b + 4 q + r)
    const uint64_t fd = (uint64_t)a.F * a.D;
    float *pg = a.part + blockIdx.x * fd, *pu = a.part + (gridDim.x + blockIdx.x) * fd, *pd = a.part + 2ull * gridDim.x * fd + (uint64_t)blockIdx.x * a.O * a.F;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const uint32_t f = slice * 32u + 16u * (i >> 2 & 1u) + 4u * (2u * c + (i >> 3)) + (i & 3u);
        if (f < a.F) {
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const uint32_t n = d * 16u + 4u * g;
                const float v[4] = {sum_g[c][d][0], sum_g[c][d][1], sum_g[c][d][2], sum_g[c][d][3]}, w[4] = {sum_u[c][d][0], sum_u[c][d][1], sum_u[c][d][2], sum_u[c][d][3]};
                store_row4(pg + (uint64_t)f * a.D + n, (int64_t)a.D - n, v);
                store_row4(pu + (uint64_t)f * a.D + n, (int64_t)a.D - n, w);
            }
        }
        const uint32_t f4 = slice * 32u + 16u * (g & 1u) + 4u * (2u * c + (g >> 1));
#pragma unroll
        for (int o = 0; o < 2; ++o) {
            const float v[4] = {sum_d[c][o][0], sum_d[c][o][1], sum_d[c][o][2], sum_d[c][o][3]};
            if (o * 16u + i < a.O) store_row4(pd + (uint64_t)(o * 16u + i) * a.F + f4, (int64_t)a.F - f4, v);
        }
    }
}

template <class E, int ACT> int launch(const NarrowGradArgs& a, uint32_t grid, hipStream_t s) {
    auto go = [&](auto db, auto one) { hipLaunchKernelGGL((k_narrow_backward<E, ACT, decltype(db)::value, decltype(one)::value>), dim3(grid), dim3(kWaves * 64), 0, s, a); };
    auto any = [&](auto db) {
        if (a.slices == kWaves) go(db, std::true_type{});
        else go(db, std::false_type{});
    };
    if (a.D <= 32u) any(std::integral_constant<int, 2>{});
    else if (a.D <= 64u) any(std::integral_constant<int, 4>{});
    else if (a.D <= 80u) go(std::integral_constant<int, 5>{}, std::true_type{});
    else go(std::integral_constant<int, 6>{}, std::true_type{});
    return check_launch("k_narrow_backward");
}

}  // namespace

// Widths whose gradients' sums fit eight waves' registers.  Against the tiles, a training pass in bf16: 146 000 rows of 72 -> 256 -> 12 245 -> 130 us, of 96 -> 33
// -> 32 141 -> 108, of 32 -> 64 -> 16 126 -> 45; 10 000 rows of 72 -> 256 -> 12 51 both; 65 rows 35 -> 32.
bool gated_grad_is_narrow(uint32_t D, uint32_t F, uint32_t O, int dtype) { return dtype != ENVIDR_F32 && D <= 96 && F <= 256 && O <= 32; }

uint32_t gated_narrow_grad_parts(uint32_t M, uint32_t D, uint32_t F) {
    const uint32_t tiles = ceil_div(M, kWaves / narrow_slices(D, F) * (uint32_t)kTeamRows);
    return tiles < 256u ? tiles : 256u;
}

int gated_narrow_backward(NarrowGradArgs a, int dtype, int activation, hipStream_t s) {
    a.slices = narrow_slices(a.D, a.F);
    const uint32_t grid = gated_narrow_grad_parts(a.M, a.D, a.F);
    if (dtype == ENVIDR_BF16) ENVIDR_FOR_ACT(activation, ACT, return (launch<__bf16, ACT>(a, grid, s)));
    ENVIDR_FOR_ACT(activation, ACT, return (launch<_Float16, ACT>(a, grid, s)));
}

}  // namespace envidr
