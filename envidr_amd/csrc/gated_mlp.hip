// The gated feed-forward block  y = h Wd^T,  h = act(g) * u,  g = x Wg^T,  u = x Wu^T,  and its gradients.
//
//   forward   k_glu_forward  g and u in one tile (a wave holds the gate and the up column of the same hidden unit), act and product in the
//                            epilogue, h stored once as the next product's operand
//             k_product      y = h Wd^T
//   backward  k_glu_backward g, u again and dh = dy Wd in one tile; dg = dh u act'(g), du = dh act(g) and h in the epilogue, from 32-bit values
//             k_product      dx = dg Wg + du Wu (one reduction over 2 F)
//             k_weight_grads dWg = dg^T x, dWu = du^T x, dWd = dy^T h: one launch, the reduction over the rows split where the results are too few
//                            to fill the chip; partial sums in fp32, added in a fixed order
// 16-bit types: h, dg and du are rounded to the type as the operands of the next product, for half its time and bytes: as two terms each they would
// double them.  It adds one rounding, as large as the result's own: relative to the result, root of the mean square, 2.3e-3 in bf16 and 2.9e-4 in fp16
// where 32-bit values between the products give 1.7e-3 and 2.1e-4.  (k_few_rows, bound by the weights' bytes, keeps 32 bits.)
// Why g and u are formed again: kept in 32 bits they cost 16 bytes a hidden unit of traffic, more than the 4 D flops of forming them while
// D is below about 800; kept in 16 bits they would cost the gradients half a bit.
//
// Operands that the core cannot read as they are (fp32: three bf16 terms; widths, pitches or addresses that are no multiples of 16 bytes) are
// laid out first by k_pack_operands.  Rows go in chunks of at most kChunkBytes of hidden-layer operands.
//
// Narrow layers go forward in one kernel (all weights in one CU's LDS: gated_narrow.hip; fp32: in its registers, gated_narrow_fp32.hip), those of the
// 16-bit types backward in another (the sums of the weights' gradients in one CU's registers: gated_narrow_grad.hip).
//
// Of few rows the weights' bytes are all there is to move: k_few_rows streams them once through registers, sixteen weight rows a workgroup, the
// reduction split over its waves.
#include "gated_mlp.hip.h"
#include "gemm_core.hip.h"

#include <type_traits>

namespace envidr {
namespace {

// ---- layout of operands ----------------------------------------------------------------------------------------------------------------
struct PackJob {
    const void* src;
    uint16_t* dst;
    int64_t ld;
    uint64_t plane;
    uint32_t rows, cols, units;     // units = padded row / 8
    uint32_t first_block;
};
struct PackJobs {
    PackJob job[5];
    uint32_t n;
    uint32_t from;                  // the launch's first block
};

// Grids that grow with the data are launched in runs: a launch holds fewer than 2^32 threads.  (Blocks that walk instead cost the sums of a
// training pass of 4096 rows, 512 -> 2048 -> 512 in bf16, 14 us for 12.)
constexpr uint32_t kMostBlocks = (1u << 31) / kBlock;
template <class Launch> int in_runs(uint32_t blocks, Launch launch) {
    for (uint32_t from = 0; from < blocks; from += kMostBlocks)
        if (int rc = launch(from, blocks - from < kMostBlocks ? blocks - from : kMostBlocks)) return rc;
    return ENVIDR_OK;
}

template <class E, class T, int NP> __global__ void __launch_bounds__(kBlock) k_pack_operands(PackJobs a) {
    const uint32_t block = a.from + blockIdx.x;
    uint32_t j = 0;
    while (j + 1 < a.n && block >= a.job[j + 1].first_block) ++j;
    const PackJob p = a.job[j];
    const uint64_t at = (uint64_t)(block - p.first_block) * kBlock + threadIdx.x;
    const uint64_t row = at / p.units;
    if (row >= p.rows) return;
    const uint32_t c0 = (uint32_t)(at % p.units) * 8u;
    const E* s = static_cast<const E*>(p.src) + row * p.ld + c0;
    float v[8];
    if (c0 + 8u <= p.cols) {
        const Pack<E, 8> x = load_pack<E, 8>(s);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f32(x.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c0 + i < p.cols ? to_f32(s[i]) : 0.0f;
    }
    uint16_t* d = p.dst + (row * p.units + at % p.units) * 8u;
    store_planes<T, NP>(d, p.plane, {v[0], v[1], v[2], v[3]});
    store_planes<T, NP>(d + 4, p.plane, {v[4], v[5], v[6], v[7]});
}

// ---- tiles -----------------------------------------------------------------------------------------------------------------------------
// The kernels below are persistent: as many workgroups as the chip holds at once walk the tiles, and the first two steps of a workgroup's next
// product are loaded under the last two of the present one, before its results are stored.

struct GluArgs {
    Operand x, wg, wu, dy, wd;
    uint32_t M, F, D, O;            // D, O: the lengths of the reductions
    uint32_t Fp;
    uint16_t *h, *dg, *du;          // [M][Fp] planes
    uint64_t plane;
    uint32_t col_tiles, tiles;
};

// The units that fill the last operand unit up (columns F .. Fp - 1) have weights of zero, which an infinity in x or dy makes NaN: they are cleared, or
// the next product would carry that into its whole row.  (fp32 operands with an infinity are NaN anyway.)
template <int NP, int B, int N> __device__ __forceinline__ void clear_behind(float (&v)[B][N][4], uint32_t f0, uint32_t F) {
    if (NP == 3 || f0 + N * 16u <= F) return;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const bool behind = f0 + j * 16u + 4u * (threadIdx.x >> 4 & 3u) + r >= F;
#pragma unroll
            for (int b = 0; b < B; ++b) v[b][j][r] = behind ? 0.0f : v[b][j][r];
        }
}

template <class T, int NP, int TM, int TF, int WM, int WN, int ACT> __global__ void __launch_bounds__(WM* WN * 64, 2) k_glu_forward(GluArgs a) {
    using P = Product<T, NP, TM, 2 * TF, WM, WN, true, true, true>;
    using Out = PlaneStore<T, NP, P::NI * 8>;
    constexpr int kStores = P::MI / Out::kBlocks * Out::kCount;
    __shared__ __attribute__((aligned(1024))) char lds_all[2 * P::kStage + WM * WN * 2048];
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_void*)lds_all, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), scratch = lds + 2 * P::kStage + wave * 2048u;
    TileWalk walk(a.tiles);
    if (!walk.valid()) return;
    typename P::Source src;
    const uint32_t n = P::steps(a.D);
    auto aim = [&](uint32_t t) { src.init(a.x, a.wg, a.wu, t / a.col_tiles * TM, t % a.col_tiles * TF, 0, a.D); };
    aim(walk.now);
    src.issue(lds);
    src.issue(lds + P::kStage);
    uint32_t stage = 0;
    for (bool fresh = true; walk.valid(); walk.now += walk.by, fresh = false) {
        const uint32_t row0 = walk.now / a.col_tiles * TM + wave / WN * (P::MI * 16u), f0 = walk.now % a.col_tiles * TF + wave % WN * (P::NI * 8u);
        const bool more = walk.more();
        f32x4 acc[P::MI][P::NI] = {};
        P::template run<kStores>(lds, P::kStage, stage, src, n, !fresh, acc, 0, [&] { if (more) aim(walk.now + walk.by); }, [&](uint32_t to) { if (more) src.issue(to); });
#pragma unroll
        for (int mi = 0; mi < P::MI; mi += Out::kBlocks) {
            float h[Out::kBlocks][P::NI / 2][4];
#pragma unroll
            for (int b = 0; b < Out::kBlocks; ++b)
#pragma unroll
                for (int j = 0; j < P::NI / 2; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        h[b][j][r] = activation_value<ACT, NP == 3>(acc[mi + b][2 * j][r]) * acc[mi + b][2 * j + 1][r];
                    }
            clear_behind<NP>(h, f0, a.F);
            Out::store(scratch, h, a.h, a.plane, a.Fp, a.M, row0 + mi * 16u, f0, a.Fp);
        }
    }
}

template <class T, int NP, int TM, int TF, int WM, int WN, int ACT> __global__ void __launch_bounds__(WM* WN * 64, 2) k_glu_backward(GluArgs a) {
    using P = Product<T, NP, TM, 2 * TF, WM, WN, true, true, true>;
    using Q = Product<T, NP, TM, TF, WM, WN, true, false, false, TF == 96 ? 128 : TF>;
    using Out = PlaneStore<T, NP, Q::NI * 16>;
    constexpr int kStores = P::MI / Out::kBlocks * Out::kCount * 3;
    __shared__ __attribute__((aligned(1024))) char lds_all[2 * P::kStage + WM * WN * 2048];
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_void*)lds_all, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), scratch = lds + 2 * P::kStage + wave * 2048u;
    TileWalk walk(a.tiles);
    if (!walk.valid()) return;
    typename P::Source src;
    typename Q::Source src_h;
    auto aim = [&](uint32_t t) { src.init(a.x, a.wg, a.wu, t / a.col_tiles * TM, t % a.col_tiles * TF, 0, a.D); };
    aim(walk.now);
    src.issue(lds);
    src.issue(lds + P::kStage);
    uint32_t stage = 0;
    for (bool fresh = true; walk.valid(); walk.now += walk.by, fresh = false) {
        const uint32_t tile_row = walk.now / a.col_tiles * TM, tile_col = walk.now % a.col_tiles * TF;
        const uint32_t row0 = tile_row + wave / WN * (P::MI * 16u), f0 = tile_col + wave % WN * (Q::NI * 16u);
        const bool more = walk.more();
        f32x4 acc[P::MI][P::NI] = {}, dh[Q::MI][Q::NI] = {};
        P::template run<kStores>(lds, P::kStage, stage, src, P::steps(a.D), !fresh, acc, 0, [&] { src_h.init(a.dy, a.wd, a.wd, tile_row, tile_col, 0, a.O); }, [&](uint32_t to) { src_h.issue(to); });
        Q::template run<0>(lds, P::kStage, stage, src_h, Q::steps(a.O), false, dh, 0, [&] { if (more) aim(walk.now + walk.by); }, [&](uint32_t to) { if (more) src.issue(to); });
#pragma unroll
        for (int mi = 0; mi < P::MI; mi += Out::kBlocks) {
            float h[Out::kBlocks][Q::NI][4], dg[Out::kBlocks][Q::NI][4], du[Out::kBlocks][Q::NI][4];
#pragma unroll
            for (int b = 0; b < Out::kBlocks; ++b)
#pragma unroll
                for (int j = 0; j < Q::NI; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float act, slope;
                        const float u = acc[mi + b][2 * j + 1][r], d = dh[mi + b][j][r];
                        activation<ACT, NP == 3>(acc[mi + b][2 * j][r], act, slope);
                        h[b][j][r] = act * u;
                        dg[b][j][r] = d * u * slope;
                        du[b][j][r] = d * act;
                    }
            clear_behind<NP>(dg, f0, a.F);
            clear_behind<NP>(du, f0, a.F);
            Out::store(scratch, h, a.h, a.plane, a.Fp, a.M, row0 + mi * 16u, f0, a.Fp);
            Out::store(scratch, dg, a.dg, a.plane, a.Fp, a.M, row0 + mi * 16u, f0, a.Fp);
            Out::store(scratch, du, a.du, a.plane, a.Fp, a.M, row0 + mi * 16u, f0, a.Fp);
        }
    }
}

struct ProductArgs {
    Operand a[2], b[2];             // phases: the reduction runs over a[0] b[0], then a[1] b[1]
    uint32_t K;
    uint32_t phases;
    void* out;
    int64_t ld;
    uint32_t M, N, col_tiles, tiles;
    bool aligned;
    uint32_t splits, per_split;     // splits > 0: each phase's reduction is cut into that many, and every part is a tile of its own whose sums
    float* part;                    // go to part [phases * splits][M][N]
};

// rows x columns results of type E: BKC: b K-contiguous (y = h Wd^T), else K-strided (dx = dg Wg + du Wu)
template <class E, class T, int NP, int TM, int TN, int WM, int WN, bool BKC> __global__ void __launch_bounds__(WM* WN * 64, 2) k_product(ProductArgs a) {
    using P = Product<T, NP, TM, TN, WM, WN, true, BKC, false>;
    using Out = ResultStore<E, P::MI, P::NI>;
    __shared__ __attribute__((aligned(1024))) char lds_all[2 * P::kStage + (Out::kWide ? 0 : WM * WN * 2048)];
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_void*)lds_all, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), scratch = lds + 2 * P::kStage + wave * 2048u;
    TileWalk walk(a.tiles * (a.splits ? a.splits * a.phases : 1u));
    if (!walk.valid()) return;
    typename P::Source src;
    struct Spot { uint32_t part, row0, col0, phase, from, to; };
    auto spot = [&](uint32_t i, uint32_t p) {
        Spot s;
        const uint32_t t = i % a.tiles;
        s.part = i / a.tiles;
        s.row0 = t / a.col_tiles * TM;
        s.col0 = t % a.col_tiles * TN;
        s.phase = a.splits ? s.part / a.splits : p;
        s.from = a.splits ? min(s.part % a.splits * a.per_split, a.K) : 0u;
        s.to = a.splits ? min(s.from + a.per_split, a.K) : a.K;
        return s;
    };
    auto aim = [&](const Spot& s) { src.init(s.phase ? a.a[1] : a.a[0], s.phase ? a.b[1] : a.b[0], a.b[0], s.row0, s.col0, s.from, s.to); };
    const uint32_t runs = a.splits ? 1u : a.phases;             // one after the other into the same sums
    Spot now = spot(walk.now, 0), next = now;
    aim(now);
    src.issue(lds);
    src.issue(lds + P::kStage);
    uint32_t stage = 0;
    for (bool fresh = true; walk.valid(); walk.now += walk.by, fresh = false) {
        const bool more = walk.more();
        f32x4 acc[P::MI][P::NI] = {};
        for (uint32_t p = 0; p < runs; ++p) {
            const bool goes_on = more || p + 1 < runs;
            P::template run<Out::kCount>(lds, P::kStage, stage, src, P::steps(now.to - now.from), !fresh && a.aligned && p == 0 && !a.splits, acc, 0,
                                         [&] { if (goes_on) { next = p + 1 < runs ? spot(walk.now, p + 1) : spot(walk.now + walk.by, 0); aim(next); } }, [&](uint32_t to) { if (goes_on) src.issue(to); });
            if (p + 1 < runs) now = next;
        }
        const uint32_t row0 = now.row0 + wave / WN * (P::MI * 16u), col0 = now.col0 + wave % WN * (P::NI * 16u);
        if (a.splits) ResultStore<float, P::MI, P::NI>::store(scratch, acc, a.part + (uint64_t)now.part * a.M * a.N, a.N, a.M, a.N, row0, col0, a.N % 4u == 0);
        else Out::store(scratch, acc, static_cast<E*>(a.out), a.ld, a.M, a.N, row0, col0, a.aligned);
        now = next;
    }
}

struct GradJob {
    Operand a, b;                   // both K-strided: result rows = a's columns
    void* out;                      // [rows][cols], dense
    float* part;                    // [splits][rows][cols] fp32, or NULL: the results go straight to `out`
    uint32_t rows, cols, col_tiles, first_tile;
    bool aligned;
};
struct GradArgs {
    GradJob job[3];
    uint32_t jobs, K, per_split, splits, tiles;     // tiles: of one split
    bool add;                       // to what `part` holds (a later chunk of rows)
};

template <class E, class T, int NP, int TM, int TN, int WM, int WN> __global__ void __launch_bounds__(WM* WN * 64, 2) k_weight_grads(GradArgs a) {
    using P = Product<T, NP, TM, TN, WM, WN, false, false, false>;
    using Part = ResultStore<float, P::MI, P::NI>;
    using Out = ResultStore<E, P::MI, P::NI>;
    __shared__ __attribute__((aligned(1024))) char lds_all[2 * P::kStage + (Out::kWide ? 0 : WM * WN * 2048)];
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_void*)lds_all, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), scratch = lds + 2 * P::kStage + wave * 2048u;
    TileWalk walk(a.tiles * a.splits);
    if (!walk.valid()) return;
    struct Spot { uint32_t split, j, row0, col0, from, to; };
    auto spot = [&](uint32_t tt) {
        Spot s;
        s.split = tt / a.tiles;
        const uint32_t t = tt % a.tiles;
        s.j = 0;
        while (s.j + 1 < a.jobs && t >= a.job[s.j + 1].first_tile) ++s.j;
        const uint32_t i = t - a.job[s.j].first_tile;
        s.row0 = i / a.job[s.j].col_tiles * TM;
        s.col0 = i % a.job[s.j].col_tiles * TN;
        s.from = min(s.split * a.per_split, a.K);
        s.to = min(s.from + a.per_split, a.K);
        return s;
    };
    typename P::Source src;
    auto aim = [&](const Spot& s) { src.init(a.job[s.j].a, a.job[s.j].b, a.job[s.j].b, s.row0, s.col0, s.from, s.to); };
    Spot now = spot(walk.now), next = now;
    aim(now);
    src.issue(lds);
    src.issue(lds + P::kStage);
    uint32_t stage = 0;
    for (; walk.valid(); walk.now += walk.by, now = next) {
        const bool more = walk.more();
        f32x4 acc[P::MI][P::NI] = {};
        P::template run<0>(lds, P::kStage, stage, src, P::steps(now.to - now.from), false, acc, 0, [&] { if (more) { next = spot(walk.now + walk.by); aim(next); } }, [&](uint32_t to) { if (more) src.issue(to); });
        const GradJob& g = a.job[now.j];
        const uint32_t row0 = now.row0 + wave / WN * (P::MI * 16u), col0 = now.col0 + wave % WN * (P::NI * 16u);
        if (!g.part) {
            Out::store(scratch, acc, static_cast<E*>(g.out), g.cols, g.rows, g.cols, row0, col0, g.aligned);
            continue;
        }
        float* part = g.part + (uint64_t)now.split * g.rows * g.cols;
        if (a.add) {
            const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
            for (int mi = 0; mi < P::MI; ++mi)
#pragma unroll
                for (int ni = 0; ni < P::NI; ++ni) {
                    const uint32_t m = row0 + mi * 16u + (lane & 15u), n = col0 + ni * 16u + 4u * (lane >> 4);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (m < g.rows && n + r < g.cols) acc[mi][ni][r] += part[(uint64_t)m * g.cols + n + r];
                }
        }
        Part::store(scratch, acc, part, g.cols, g.rows, g.cols, row0, col0, g.cols % 4u == 0);
    }
}

struct SumJob {
    const float* part;              // [splits][n / cols][cols]
    void* out;
    uint64_t n;
    uint32_t first_block, cols;
    int64_t ld;                     // of out
};
struct SumArgs {
    SumJob job[3];
    uint32_t jobs, splits;
    uint32_t from;                  // the launch's first block
};
// SHARE threads add up a result's parts, every SHARE-th each, and the first adds theirs
template <class E, int SHARE> __global__ void __launch_bounds__(kBlock) k_sum_splits(SumArgs a) {
    constexpr uint32_t kResults = kBlock / SHARE;
    const uint32_t block = a.from + blockIdx.x;
    uint32_t j = 0;
    while (j + 1 < a.jobs && block >= a.job[j + 1].first_block) ++j;
    const SumJob& s = a.job[j];
    const uint64_t i = (uint64_t)(block - s.first_block) * kResults + threadIdx.x % kResults;
    float v = 0;
    if (i < s.n) {
#pragma unroll 8
        for (uint32_t k = threadIdx.x / kResults; k < a.splits; k += SHARE) v += s.part[k * s.n + i];
    }
    if constexpr (SHARE > 1) {
        __shared__ float shared[kBlock];
        shared[threadIdx.x] = v;
        __syncthreads();
        if (threadIdx.x >= kResults) return;
#pragma unroll
        for (int k = 1; k < SHARE; ++k) v += shared[k * kResults + threadIdx.x];
    }
    if (i < s.n) static_cast<E*>(s.out)[(int64_t)(i / s.cols) * s.ld + (int64_t)(i % s.cols)] = from_f32<E>(v);
}

// ---- few rows --------------------------------------------------------------------------------------------------------------------------
struct FewArgs {
    const void *a, *w, *w2;
    void* out;
    int64_t lda, ldw, ldw2, ldo;
    uint32_t M, K, N;
};
constexpr int kFewWaves = 8;

// Sixteen weight rows (of one or of both matrices) x all rows of a (MT blocks of 16); every wave takes every kFewWaves-th step of the reduction.
// GLU: a is x, the result h in 32 bits; else a is that h, for the 16-bit matrix cores as two terms of the type (rounded, and what the rounding
// left): the weights' bytes are what counts here, and y then has its own rounding only.
template <class E, int ACT, bool GLU, int MT> __global__ void __launch_bounds__(kFewWaves * 64) k_few_rows(FewArgs f) {
    using A = typename std::conditional<GLU, E, float>::type;
    using Out = typename std::conditional<GLU, float, E>::type;
    constexpr int W = 16 / sizeof(E);                    // elements of a lane's 16 bytes of weights
    constexpr uint32_t kStep = 4 * W;                    // k of a wave's step: four lane groups
    constexpr int kMats = GLU ? 2 : 1;
    __shared__ f32x4 part[kMats][kFewWaves][64];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, i = lane & 15u, n0 = blockIdx.x * 16u;
    const A* a[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) a[t] = static_cast<const A*>(f.a) + (int64_t)min(16u * t + i, f.M - 1u) * f.lda;
    const uint32_t wr = min(n0 + i, f.N - 1u);
    const E* w[kMats];
    w[0] = static_cast<const E*>(f.w) + (int64_t)wr * f.ldw;
    if constexpr (GLU) w[1] = static_cast<const E*>(f.w2) + (int64_t)wr * f.ldw2;
    f32x4 acc[kMats][MT] = {};
    auto fetch = [&](const auto* p, uint32_t k) {
        using P = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
        if (k + W <= f.K) return load_pack<P, W>(p + k);
        Pack<P, W> v;
#pragma unroll
        for (int q = 0; q < W; ++q) v.v[q] = k + q < f.K ? p[k + q] : from_f32<P>(0.0f);
        return v;
    };
    // kAhead of a wave's steps at a time: their loads are all out before the first is waited for (one row, 1024 -> 4096 -> 1024: bf16 18 us, fp32 26;
    // a step at a time 20 and 31)
    constexpr int kAhead = MT == 1 ? 4 : 2;
    for (uint32_t first = wave * kStep; first < f.K; first += kAhead * kFewWaves * kStep) {
        Pack<E, W> y[kAhead][kMats];
        Pack<A, W> x[kAhead][MT];
#pragma unroll
        for (int s = 0; s < kAhead; ++s) {
            const uint32_t k0 = first + s * (kFewWaves * kStep), k = k0 + g * W;
            if (k0 + kStep <= f.K) {
#pragma unroll
                for (int m = 0; m < kMats; ++m) y[s][m] = load_pack<E, W>(w[m] + k);
#pragma unroll
                for (int t = 0; t < MT; ++t) x[s][t] = load_pack<A, W>(a[t] + k);
            } else if (k0 < f.K) {
#pragma unroll
                for (int m = 0; m < kMats; ++m) y[s][m] = fetch(w[m], k);
#pragma unroll
                for (int t = 0; t < MT; ++t) x[s][t] = fetch(a[t], k);
            }
        }
#pragma unroll
        for (int s = 0; s < kAhead; ++s) {
            if (first + s * (kFewWaves * kStep) >= f.K) break;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                if constexpr (sizeof(E) == 4) {
#pragma unroll
                    for (int m = 0; m < kMats; ++m)
#pragma unroll
                        for (int q = 0; q < 4; ++q) acc[m][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(y[s][m].v[q], x[s][t].v[q], acc[m][t], 0, 0, 0);
                } else if constexpr (GLU) {
#pragma unroll
                    for (int m = 0; m < kMats; ++m) acc[m][t] = mfma16<E>(__builtin_bit_cast(s16x8, y[s][m]), __builtin_bit_cast(s16x8, x[s][t]), acc[m][t]);
                } else {
                    Pack<E, W> hi, lo;
#pragma unroll
                    for (int q = 0; q < W; ++q) {
                        hi.v[q] = from_f32<E>(x[s][t].v[q]);
                        const float rounded = to_f32(hi.v[q]);
                        lo.v[q] = from_f32<E>(__builtin_isinf(rounded) ? 0.0f : x[s][t].v[q] - rounded);       // (inf - inf would be NaN)
                    }
                    acc[0][t] = mfma16<E>(__builtin_bit_cast(s16x8, y[s][0]), __builtin_bit_cast(s16x8, lo), acc[0][t]);
                    acc[0][t] = mfma16<E>(__builtin_bit_cast(s16x8, y[s][0]), __builtin_bit_cast(s16x8, hi), acc[0][t]);
                }
            }
        }
    }
    const uint32_t n = n0 + 4u * g;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        // (block t's sums are added up by wave t)
#pragma unroll
        for (int m = 0; m < kMats; ++m) part[m][wave][lane] = acc[m][t];
        __syncthreads();
        const uint32_t row = 16u * t + i;
        if (wave == (uint32_t)t && row < f.M) {
            f32x4 sum[kMats] = {};
#pragma unroll
            for (int m = 0; m < kMats; ++m)
#pragma unroll
                for (int q = 0; q < kFewWaves; ++q) sum[m] += part[m][q][lane];
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (GLU) v[r] = activation_value<ACT, true>(sum[0][r]) * sum[1][r];
                else v[r] = sum[0][r];
            }
            store_row4(static_cast<Out*>(f.out) + (int64_t)row * f.ldo + n, (int64_t)f.N - n, v);
        }
        if (t + 1 < MT) __syncthreads();
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------
constexpr uint64_t kChunkBytes = 2ull << 30;    // of hidden-layer operands at a time
constexpr uint32_t kMaxChunk = 1u << 22;        // rows (tile numbers stay within 32 bits at any width)
constexpr uint32_t kMaxWidth = 1u << 20;

// Rows that go forward through k_few_rows.  512 -> 2048 -> 512 and 1024 -> 4096 -> 1024 in bf16: 17 and 23 us at 16 rows, 21 and 32 at 32, 31 and 50 at
// 64, where the tiles take 22 and 31.  256 -> 1000 -> 250 in fp32: 26 us at 64 rows, the tiles (with their three terms to lay out) 37.
uint32_t few_rows(int dtype) { return dtype == ENVIDR_F32 ? 64u : 32u; }

uint32_t pad8(uint32_t v) { return (v + 7u) / 8u * 8u; }

// where everything lies in the workspace, in bytes
struct Plan {
    uint32_t np, Dp, Fp, Op, chunk;
    uint32_t splits, per_split;
    bool large_grads;
    uint32_t product_splits, product_per_split;     // of y's reduction, or of either of dx's
    uint64_t product_part;
    uint64_t x, dy, wg, wu, wd, h, dg, du, part, bytes;
};

// Tiles.  Large: 256 x 256 by eight waves, one workgroup a CU -- LDS reads take 3/4 of the products' time where 128 x 128 by four waves takes
// all of it (32 768 x 4096 x 1024, bf16: 1060 against 780 TFLOP/s).  The three terms of fp32 fill the LDS with 256 x 128, and six products a
// pair of reads leave the reads' share below half.  Small where the large tiles are fewer than 3/4 of the CUs: bf16 training pass of 4096 rows,
// 512 -> 2048 -> 512: 198 us so and 279 with large tiles throughout; forward of 16 384 rows, 1024 -> 1024 -> 1024: 98 us with large ones, 113 with small.
constexpr uint32_t kCus = 256, kEnoughTiles = 192;
struct TileSize {
    uint32_t m, n;
};
uint64_t tiles_of(uint64_t rows, uint64_t cols, TileSize t) { return (rows + t.m - 1) / t.m * ((cols + t.n - 1) / t.n); }
constexpr TileSize product_tile(uint32_t np, bool large) { return large ? (np == 1 ? TileSize{256, 256} : TileSize{256, 128}) : TileSize{128, 128}; }
bool large_product(uint64_t rows, uint64_t cols, uint32_t np) { return tiles_of(rows, cols, product_tile(np, true)) >= kEnoughTiles; }
uint64_t grad_tiles(uint32_t D, uint32_t F, uint32_t O, TileSize t) { return 2 * tiles_of(F, D, t) + tiles_of(O, F, t); }
// workgroups a CU holds: by the LDS of two stages of a (rows + cols)-wide tile and the waves' 2 KiB
constexpr uint32_t per_cu(int np, int rows, int cols, int waves) {
    return 2 * (2 * np * (rows + cols) * (np == 1 ? 64 : 32) * 2 + waves * 2048) <= 160 * 1024 ? 2u : 1u;
}
// workgroups: as many as are resident at once, in whole rounds of the XCDs
uint32_t grid_of(uint64_t tiles, uint32_t per_cu) {
    const uint64_t all = (tiles + 7) / 8 * 8, most = (uint64_t)kCus * per_cu;
    return (uint32_t)(all < most ? all : most);
}

// Few tiles and a long reduction (a small batch through a wide layer): a step of the reduction costs a workgroup about 0.7 us of latency however
// few workgroups there are, so each reduction is cut until the tiles' parts fill the chip, in parts of four steps at least.  From twelve
// steps on that gains more than the launch that adds the parts up costs (500 x 1000 outputs over 4000: 44 -> 15 us).
uint32_t product_splits(uint64_t rows, uint64_t cols, uint32_t k, uint32_t phases, uint32_t np) {
    if (large_product(rows, cols, np)) return 0;
    const uint32_t steps = ceil_div(k, np == 1 ? 64u : 32u);
    const uint64_t tiles = tiles_of(rows, cols, product_tile(np, false)) * phases, slots = kCus * (np == 1 ? 2u : 1u);
    if (tiles * 2 > slots || steps * phases < 12u) return 0;
    const uint64_t fill = slots / tiles, can = steps / 4u ? steps / 4u : 1u;
    const uint64_t splits = fill < can ? fill : can;
    return splits * phases > 1 ? (uint32_t)splits : 0u;
}

Plan make_plan(uint32_t M, uint32_t D, uint32_t F, uint32_t O, int dtype, bool backward) {
    Plan p{};
    p.np = dtype == ENVIDR_F32 ? 3u : 1u;
    p.Dp = pad8(D);
    p.Fp = pad8(F);
    p.Op = pad8(O);
    const uint64_t row = 2ull * p.np * p.Fp * (backward ? 3u : 1u);
    const uint64_t most = kChunkBytes / row / 256u * 256u;
    p.chunk = (uint32_t)(most < 256u ? 256u : (most < kMaxChunk ? most : kMaxChunk));
    if (p.chunk > M) p.chunk = M;
    if (!backward && M <= few_rows(dtype)) {
        p.h = 0;
        p.bytes = round_up64(4ull * M * p.Fp, 256);
        return p;
    }
    if (!backward && gated_is_narrow(D, F, O, dtype)) {
        p.bytes = 16;
        return p;
    }
    if (backward && gated_grad_is_narrow(D, F, O, dtype)) {
        p.splits = gated_narrow_grad_parts(M, D, F);
        p.bytes = 4ull * p.splits * (2ull * F * D + (uint64_t)O * F);
        return p;
    }
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) { const uint64_t here = at; at += round_up64(bytes, 256); return here; };
    p.wg = take(2ull * p.np * F * p.Dp);
    p.wu = take(2ull * p.np * F * p.Dp);
    p.wd = take(2ull * p.np * O * p.Fp);
    p.x = take(2ull * p.np * p.chunk * p.Dp);
    p.h = take(2ull * p.np * p.chunk * p.Fp);
    const uint32_t cols = backward ? D : O, phases = backward ? 2u : 1u;
    if (p.chunk == M) p.product_splits = product_splits(M, cols, F, phases, p.np);
    if (p.product_splits) {
        p.product_per_split = (uint32_t)round_up64(ceil_div(F, p.product_splits), 64);
        p.product_splits = ceil_div(F, p.product_per_split);
        p.product_part = take(4ull * p.product_splits * phases * M * cols);
    }
    if (backward) {
        p.dy = take(2ull * p.np * p.chunk * p.Op);
        p.dg = take(2ull * p.np * p.chunk * p.Fp);
        p.du = take(2ull * p.np * p.chunk * p.Fp);
        // The rows' reduction is split where the results alone do not fill the chip.  Of the numbers of parts (of 512 rows at least) the one
        // whose rounds of tiles cost least, with what its partial sums cost to write and read again: in 1e-9 ms, a round of the products at
        // about 1000 TFLOP/s and a result's 8 bytes at 4 TB/s.
        const double results = 2.0 * F * D + (double)O * F, per_part = results * 2e-3;
        const uint32_t can = ceil_div(p.chunk, 512u), most_parts = can < 64u ? can : 64u;
        double best = 0;
        for (int large = 0; large < 2; ++large) {
            const TileSize tile = product_tile(p.np, large);
            const double tiles = (double)grad_tiles(D, F, O, tile), slots = kCus * (large || p.np > 1 ? 1.0 : 2.0);
            const double one_tile = 2.0 * p.chunk * tile.m * tile.n * (p.np == 3 ? 6 : 1) * slots / (large ? 1000.0 : 750.0);          // all rows of it, on its slot
            for (uint32_t s = 1; s <= most_parts; ++s) {
                const double cost = __builtin_ceil(tiles * s / slots) * one_tile / s + (s > 1 ? s * per_part : 0.0);
                if (best == 0 || cost < best) {
                    best = cost;
                    p.large_grads = large;
                    p.splits = s;
                }
            }
        }
        p.per_split = (uint32_t)round_up64(ceil_div(p.chunk, p.splits), 64);
        p.splits = ceil_div(p.chunk, p.per_split);
        if (p.splits > 1 || p.chunk < M) p.part = take(4ull * p.splits * (2ull * F * D + (uint64_t)O * F));
    }
    p.bytes = at;
    return p;
}

struct Weights {
    const void *wg, *wu, *wd;
    int64_t lg, lu, ldn;
};

// can the core read it as it is: 16-byte rows of whole units, one behind the other (it bounds a tile by its rows times the pitch, which cuts rows
// that overlap or repeat)
bool readable(const void* p, int64_t ld, uint32_t cols, int dtype) {
    return dtype != ENVIDR_F32 && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0 && cols % 8 == 0 && ld >= cols;
}

struct Packer {
    PackJobs jobs{};
    uint32_t blocks = 0;
    int dtype;
    uint32_t np;
    // the operand for [rows, cols] at src: the tensor itself, or its place in the workspace and a job
    Operand add(const void* src, int64_t ld, uint32_t rows, uint32_t cols, void* place, bool k_strided) {
        const uint32_t units = pad8(cols) / 8u;
        Operand o;
        o.ext = k_strided ? units * 8u : rows;
        if (readable(src, ld, cols, dtype)) {
            o.p = static_cast<const uint16_t*>(src);
            o.plane = 0;
            o.ld = (uint32_t)ld;
            return o;
        }
        o.p = static_cast<uint16_t*>(place);
        o.ld = units * 8u;
        o.plane = (uint64_t)rows * o.ld;
        PackJob& j = jobs.job[jobs.n++];
        j.src = src;
        j.dst = static_cast<uint16_t*>(place);
        j.ld = ld;
        j.plane = o.plane;
        j.rows = rows;
        j.cols = cols;
        j.units = units;
        j.first_block = blocks;
        blocks += (uint32_t)(((uint64_t)rows * units + kBlock - 1) / kBlock);
        return o;
    }
    template <class E, class T, int NP> int launch(hipStream_t s) {
        return in_runs(blocks, [&](uint32_t from, uint32_t n) {
            jobs.from = from;
            hipLaunchKernelGGL((k_pack_operands<E, T, NP>), dim3(n), dim3(kBlock), 0, s, jobs);
            return check_launch("k_pack_operands");
        });
    }
};

Operand hidden(const uint16_t* p, uint32_t Fp, uint32_t rows, uint64_t plane, bool k_strided) {
    return {p, plane, Fp, k_strided ? Fp : rows};
}

template <class E> struct Terms { using T = E; static constexpr int NP = 1; };
template <> struct Terms<float> { using T = __bf16; static constexpr int NP = 3; };

template <class E, int TM, int TN, int WM, int WN, bool BKC> int launch_product_as(ProductArgs a, hipStream_t s) {
    using T = typename Terms<E>::T;
    constexpr int NP = Terms<E>::NP;
    a.col_tiles = ceil_div(a.N, (uint32_t)TN);
    a.tiles = ceil_div(a.M, (uint32_t)TM) * a.col_tiles;
    hipLaunchKernelGGL((k_product<E, T, NP, TM, TN, WM, WN, BKC>), dim3(grid_of((uint64_t)a.tiles * (a.splits ? a.splits * a.phases : 1u), per_cu(NP, TM, TN, WM * WN))), dim3(WM * WN * 64), 0, s, a);
    return check_launch("k_product");
}
bool whole_units(const void* p, int64_t ld, uint32_t cols, uint32_t size) {
    const uint32_t unit = 16u / size;
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % unit == 0 && cols % unit == 0;
}
// adds up parts: `add` fills in where they lie and where their sums go
struct Sums {
    SumArgs a{};
    uint32_t share, blocks = 0;
    explicit Sums(uint32_t splits) {
        a.splits = splits;
        // Many parts of few results: four threads a result (256 parts of 40 k results 15 -> 8 us); few parts of many results: one (4 parts of
        // 12.6 M results 67 us, 110 with four).
        share = splits >= 8u ? 4u : 1u;
    }
    void add(const float* part, void* out, uint64_t rows, uint32_t cols, int64_t ld) {
        const uint64_t n = rows * cols, results = kBlock / share;
        a.job[a.jobs++] = {part, out, n, blocks, cols, ld};
        blocks += (uint32_t)((n + results - 1) / results);
    }
    template <class E> int launch(hipStream_t s) {
        return in_runs(blocks, [&](uint32_t from, uint32_t n) {
            a.from = from;
            if (share == 4u) hipLaunchKernelGGL((k_sum_splits<E, 4>), dim3(n), dim3(kBlock), 0, s, a);
            else hipLaunchKernelGGL((k_sum_splits<E, 1>), dim3(n), dim3(kBlock), 0, s, a);
            return check_launch("k_sum_splits");
        });
    }
};
// the weights' gradients from their parts, which lie one behind the other
template <class E> int sum_weight_grads(const float* part, uint32_t splits, uint32_t D, uint32_t F, uint32_t O, void* dwg, void* dwu, void* dwd, hipStream_t s) {
    const uint64_t fd = (uint64_t)splits * F * D;
    Sums u(splits);
    if (dwg) u.add(part, dwg, F, D, D);
    if (dwu) u.add(part + fd, dwu, F, D, D);
    if (dwd) u.add(part + 2 * fd, dwd, O, F, F);
    return u.template launch<E>(s);
}
template <class E, bool BKC> int launch_product(ProductArgs a, const Plan& p, char* ws, hipStream_t s) {
    constexpr int NP = Terms<E>::NP;
    a.aligned = whole_units(a.out, a.ld, a.N, sizeof(E));
    if (p.product_splits) {
        a.splits = p.product_splits;
        a.per_split = p.product_per_split;
        a.part = reinterpret_cast<float*>(ws + p.product_part);
        if (int rc = launch_product_as<E, 128, 128, 2, 2, BKC>(a, s)) return rc;
        Sums u(a.splits * a.phases);
        u.add(a.part, a.out, a.M, a.N, a.ld);
        return u.template launch<E>(s);
    }
    if (!large_product(a.M, a.N, NP)) return launch_product_as<E, 128, 128, 2, 2, BKC>(a, s);
    if constexpr (NP == 1) return launch_product_as<E, 256, 256, 2, 4, BKC>(a, s);
    else return launch_product_as<E, 256, 128, 4, 2, BKC>(a, s);
}

template <class E, int ACT, int TM, int TF, int WM, int WN> int launch_glu_forward_as(GluArgs a, hipStream_t s) {
    using T = typename Terms<E>::T;
    constexpr int NP = Terms<E>::NP;
    a.col_tiles = ceil_div(a.F, (uint32_t)TF);
    a.tiles = ceil_div(a.M, (uint32_t)TM) * a.col_tiles;
    hipLaunchKernelGGL((k_glu_forward<T, NP, TM, TF, WM, WN, ACT>), dim3(grid_of(a.tiles, per_cu(NP, TM, 2 * TF, WM * WN))), dim3(WM * WN * 64), 0, s, a);
    return check_launch("k_glu_forward");
}
template <class E, int ACT> int launch_glu_forward(const GluArgs& a, hipStream_t s) {
    constexpr int NP = Terms<E>::NP;
    if (!large_product(a.M, 2ull * a.F, NP)) return launch_glu_forward_as<E, ACT, 128, 64, 2, 2>(a, s);
    if constexpr (NP == 1) return launch_glu_forward_as<E, ACT, 256, 128, 2, 4>(a, s);
    else return launch_glu_forward_as<E, ACT, 256, 64, 4, 2>(a, s);
}

template <class E, int ACT, int TM, int TF, int WM, int WN> int launch_glu_backward_as(GluArgs a, hipStream_t s) {
    using T = typename Terms<E>::T;
    constexpr int NP = Terms<E>::NP;
    a.col_tiles = ceil_div(a.F, (uint32_t)TF);
    a.tiles = ceil_div(a.M, (uint32_t)TM) * a.col_tiles;
    hipLaunchKernelGGL((k_glu_backward<T, NP, TM, TF, WM, WN, ACT>), dim3(grid_of(a.tiles, per_cu(NP, TM, 2 * TF, WM * WN))), dim3(WM * WN * 64), 0, s, a);
    return check_launch("k_glu_backward");
}
// (three accumulators a hidden unit: half the columns of the other products)
template <class E, int ACT> int launch_glu_backward(const GluArgs& a, hipStream_t s) {
    constexpr int NP = Terms<E>::NP;
    if constexpr (NP == 1) {
        if (tiles_of(a.M, a.F, {256, 96}) >= kEnoughTiles) return launch_glu_backward_as<E, ACT, 256, 96, 4, 2>(a, s);
        return launch_glu_backward_as<E, ACT, 128, 64, 2, 2>(a, s);
    } else {
        return launch_glu_backward_as<E, ACT, 256, 64, 4, 2>(a, s);
    }
}

template <class E, int TM, int TN, int WM, int WN> int launch_weight_grads_as(const GradArgs& a, hipStream_t s) {
    using T = typename Terms<E>::T;
    constexpr int NP = Terms<E>::NP;
    hipLaunchKernelGGL((k_weight_grads<E, T, NP, TM, TN, WM, WN>), dim3(grid_of((uint64_t)a.tiles * a.splits, per_cu(NP, TM, TN, WM * WN))), dim3(WM * WN * 64), 0, s, a);
    return check_launch("k_weight_grads");
}
template <class E> int launch_weight_grads(const GradArgs& a, bool large, hipStream_t s) {
    constexpr int NP = Terms<E>::NP;
    if (!large) return launch_weight_grads_as<E, 128, 128, 2, 2>(a, s);
    if constexpr (NP == 1) return launch_weight_grads_as<E, 256, 256, 2, 4>(a, s);
    else return launch_weight_grads_as<E, 256, 128, 4, 2>(a, s);
}

template <class E> int forward(const void* x, int64_t ldx, const Weights& w, uint32_t M, uint32_t D, uint32_t F, uint32_t O, int dtype, int act,
                               void* y, int64_t ldy, char* ws, hipStream_t s) {
    using T = typename Terms<E>::T;
    constexpr int NP = Terms<E>::NP;
    const Plan p = make_plan(M, D, F, O, dtype, false);
    if (M <= few_rows(dtype)) {
        const FewArgs f{x, w.wg, w.wu, ws, ldx, w.lg, w.lu, (int64_t)p.Fp, M, D, F}, d{ws, w.wd, nullptr, y, (int64_t)p.Fp, w.ldn, 0, ldy, M, F, O};
        auto go = [&](auto mt) {
            constexpr int MT = decltype(mt)::value;
            ENVIDR_FOR_ACT(act, ACT, hipLaunchKernelGGL((k_few_rows<E, ACT, true, MT>), dim3(ceil_div(F, 16u)), dim3(kFewWaves * 64), 0, s, f));
            if (int rc = check_launch("k_few_rows")) return rc;
            hipLaunchKernelGGL((k_few_rows<E, ENVIDR_ACT_SILU, false, MT>), dim3(ceil_div(O, 16u)), dim3(kFewWaves * 64), 0, s, d);
            return check_launch("k_few_rows");
        };
        if (M <= 16) return go(std::integral_constant<int, 1>{});
        if constexpr (sizeof(E) == 4)
            if (M > 32) return go(std::integral_constant<int, 4>{});
        return go(std::integral_constant<int, 2>{});
    }
    if (gated_is_narrow(D, F, O, dtype)) return gated_narrow_forward({x, w.wg, w.wu, w.wd, y, ldx, w.lg, w.lu, w.ldn, ldy, M, D, F, O}, dtype, act, s);
    Operand owg{}, owu{}, owd{};
    for (uint32_t m0 = 0; m0 < M; m0 += p.chunk) {
        const uint32_t rows = M - m0 < p.chunk ? M - m0 : p.chunk;
        Packer pk;
        pk.dtype = dtype;
        pk.np = NP;
        if (m0 == 0) {
            owg = pk.add(w.wg, w.lg, F, D, ws + p.wg, false);
            owu = pk.add(w.wu, w.lu, F, D, ws + p.wu, false);
            owd = pk.add(w.wd, w.ldn, O, F, ws + p.wd, false);
        }
        const Operand ox = pk.add(static_cast<const E*>(x) + (int64_t)m0 * ldx, ldx, rows, D, ws + p.x, false);
        if (int rc = pk.template launch<E, T, NP>(s)) return rc;
        GluArgs a{};
        a.x = ox; a.wg = owg; a.wu = owu;
        a.M = rows; a.F = F; a.D = p.Dp; a.Fp = p.Fp;
        a.h = reinterpret_cast<uint16_t*>(ws + p.h);
        a.plane = (uint64_t)p.chunk * p.Fp;
        ENVIDR_FOR_ACT(act, ACT, if (int rc = (launch_glu_forward<E, ACT>(a, s))) return rc);
        ProductArgs q{};
        q.a[0] = hidden(a.h, p.Fp, rows, a.plane, false);
        q.b[0] = owd;
        q.K = p.Fp; q.phases = 1;
        q.out = static_cast<E*>(y) + (int64_t)m0 * ldy; q.ld = ldy; q.M = rows; q.N = O;
        if (int rc = launch_product<E, true>(q, p, ws, s)) return rc;
    }
    return ENVIDR_OK;
}

template <class E> int backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const Weights& w, uint32_t M, uint32_t D, uint32_t F, uint32_t O,
                                int dtype, int act, void* dx, int64_t lddx, void* dwg, void* dwu, void* dwd, char* ws, hipStream_t s) {
    using T = typename Terms<E>::T;
    constexpr int NP = Terms<E>::NP;
    const Plan p = make_plan(M, D, F, O, dtype, true);
    if constexpr (NP == 1) {
        if (gated_grad_is_narrow(D, F, O, dtype)) {
            float* parts = reinterpret_cast<float*>(ws);
            const bool want_w = dwg || dwu || dwd;
            if (!dx && !want_w) return ENVIDR_OK;
            if (int rc = gated_narrow_backward({dy, x, w.wg, w.wu, w.wd, dx, parts, lddy, ldx, w.lg, w.lu, w.ldn, lddx, M, D, F, O, 0, want_w}, dtype, act, s)) return rc;
            return want_w ? sum_weight_grads<E>(parts, p.splits, D, F, O, dwg, dwu, dwd, s) : ENVIDR_OK;
        }
    }
    Operand owg{}, owu{}, owd{};
    float* part = p.part ? reinterpret_cast<float*>(ws + p.part) : nullptr;
    auto strided = [](Operand o, uint32_t ext) { o.ext = ext; return o; };
    for (uint32_t m0 = 0; m0 < M; m0 += p.chunk) {
        const uint32_t rows = M - m0 < p.chunk ? M - m0 : p.chunk;
        Packer pk;
        pk.dtype = dtype;
        pk.np = NP;
        if (m0 == 0) {
            owg = pk.add(w.wg, w.lg, F, D, ws + p.wg, false);
            owu = pk.add(w.wu, w.lu, F, D, ws + p.wu, false);
            owd = pk.add(w.wd, w.ldn, O, F, ws + p.wd, true);
        }
        const Operand ox = pk.add(static_cast<const E*>(x) + (int64_t)m0 * ldx, ldx, rows, D, ws + p.x, false);
        const Operand ody = pk.add(static_cast<const E*>(dy) + (int64_t)m0 * lddy, lddy, rows, O, ws + p.dy, false);
        if (int rc = pk.template launch<E, T, NP>(s)) return rc;
        GluArgs a{};
        a.x = ox; a.wg = owg; a.wu = owu; a.dy = ody; a.wd = owd;
        a.M = rows; a.F = F; a.D = p.Dp; a.Fp = p.Fp;
        a.O = O;                        // (the K-strided weights have O rows and no padding behind them)
        a.h = reinterpret_cast<uint16_t*>(ws + p.h);
        a.dg = reinterpret_cast<uint16_t*>(ws + p.dg);
        a.du = reinterpret_cast<uint16_t*>(ws + p.du);
        a.plane = (uint64_t)p.chunk * p.Fp;
        ENVIDR_FOR_ACT(act, ACT, if (int rc = (launch_glu_backward<E, ACT>(a, s))) return rc);
        if (dx) {
            ProductArgs q{};
            q.a[0] = hidden(a.dg, p.Fp, rows, a.plane, false);
            q.a[1] = hidden(a.du, p.Fp, rows, a.plane, false);
            q.b[0] = strided(owg, p.Dp);
            q.b[1] = strided(owu, p.Dp);
            q.K = F; q.phases = 2;
            q.out = static_cast<E*>(dx) + (int64_t)m0 * lddx; q.ld = lddx; q.M = rows; q.N = D;
            if (int rc = launch_product<E, false>(q, p, ws, s)) return rc;
        }
        GradArgs g{};
        auto job = [&](Operand l, Operand r, void* out, uint64_t part_at, uint32_t n_rows, uint32_t n_cols) {
            if (!out) return;
            GradJob& j = g.job[g.jobs++];
            j.a = l; j.b = r; j.out = out; j.part = part ? part + part_at : nullptr;
            const TileSize tile = product_tile(NP, p.large_grads);
            j.rows = n_rows; j.cols = n_cols; j.col_tiles = ceil_div(n_cols, tile.n);
            j.first_tile = g.tiles;
            j.aligned = whole_units(out, n_cols, n_cols, sizeof(E));
            g.tiles += ceil_div(n_rows, tile.m) * j.col_tiles;
        };
        const uint64_t fd = (uint64_t)p.splits * F * D;
        job(hidden(a.dg, p.Fp, rows, a.plane, true), strided(ox, p.Dp), dwg, 0, F, D);
        job(hidden(a.du, p.Fp, rows, a.plane, true), strided(ox, p.Dp), dwu, fd, F, D);
        job(strided(ody, p.Op), hidden(a.h, p.Fp, rows, a.plane, true), dwd, 2 * fd, O, F);
        if (g.jobs) {
            g.K = rows; g.per_split = p.per_split; g.splits = p.splits; g.add = m0 > 0;
            if (int rc = launch_weight_grads<E>(g, p.large_grads, s)) return rc;
        }
    }
    if (part && (dwg || dwu || dwd)) return sum_weight_grads<E>(part, p.splits, D, F, O, dwg, dwu, dwd, s);
    return ENVIDR_OK;
}

// n zeros; a launch holds fewer than 2^32 threads, so each walks
__global__ void __launch_bounds__(kBlock) k_zero(uint16_t* p, uint64_t n) {
    for (uint64_t i = (uint64_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (uint64_t)gridDim.x * kBlock) p[i] = 0;
}

int gated_checks(const char* what, uint32_t M, uint32_t D, uint32_t F, uint32_t O, int dtype, int activation) {
    ENVIDR_REQUIRE(dtype_ok(dtype), "%s: unknown dtype %d", what, dtype);
    ENVIDR_REQUIRE(activation >= ENVIDR_ACT_SILU && activation <= ENVIDR_ACT_SIGMOID, "%s: unknown activation %d", what, activation);
    ENVIDR_REQUIRE(D >= 1 && F >= 1 && O >= 1 && D <= kMaxWidth && F <= kMaxWidth && O <= kMaxWidth, "%s: widths D=%u, F=%u, O=%u must be in 1 .. %u", what, D, F, O, kMaxWidth);
    ENVIDR_REQUIRE(M <= 0x7FFFFF00u && (uint64_t)F * D <= 1ull << 32 && (uint64_t)O * F <= 1ull << 32, "%s: M=%u rows or a weight matrix of more than 2^32 elements", what, M);
    return ENVIDR_OK;
}

int workspace_checks(const char* what, const void* workspace, uint64_t have, uint64_t need) {
    ENVIDR_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && have >= need, "%s: workspace of %llu bytes, %llu needed (16-byte aligned)", what,
                   (unsigned long long)have, (unsigned long long)need);
    return ENVIDR_OK;
}

}  // namespace
}  // namespace envidr

using namespace envidr;

extern "C" {

uint64_t envidr_gated_mlp_workspace_bytes(uint32_t M, uint32_t D, uint32_t F, uint32_t O, int dtype, int backward) {
    if (M == 0 || gated_checks("gated_mlp", M, D, F, O, dtype, ENVIDR_ACT_SILU)) return 0;
    return make_plan(M, D, F, O, dtype, backward != 0).bytes;
}

int envidr_gated_mlp_forward(const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate, const void* w_up, int64_t ld_up,
                             const void* w_down, int64_t ld_down, uint32_t M, uint32_t D, uint32_t F, uint32_t O, int dtype, int activation,
                             void* y, int64_t ldy, void* workspace, uint64_t workspace_bytes, envidr_stream_t stream) {
    if (int rc = gated_checks("gated_mlp_forward", M, D, F, O, dtype, activation)) return rc;
    if (M == 0) return ENVIDR_OK;
    ENVIDR_REQUIRE(x && w_gate && w_up && w_down && y, "gated_mlp_forward: null pointer");
    const int64_t most = 1ll << 21;
    ENVIDR_REQUIRE(ldx >= 0 && ld_gate >= 0 && ld_up >= 0 && ld_down >= 0 && ldx <= most && ld_gate <= most && ld_up <= most && ld_down <= most,
                   "gated_mlp_forward: a row pitch is negative or above 2^21");
    ENVIDR_REQUIRE(ldy >= O && ldy <= most, "gated_mlp_forward: ldy=%lld < O=%u, or above 2^21", (long long)ldy, O);
    if (int rc = workspace_checks("gated_mlp_forward", workspace, workspace_bytes, envidr_gated_mlp_workspace_bytes(M, D, F, O, dtype, 0))) return rc;
    const Weights w{w_gate, w_up, w_down, ld_gate, ld_up, ld_down};
    ENVIDR_FOR_DTYPE(dtype, E, return forward<E>(x, ldx, w, M, D, F, O, dtype, activation, y, ldy, static_cast<char*>(workspace), as_stream(stream)));
}

int envidr_gated_mlp_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w_gate, int64_t ld_gate,
                              const void* w_up, int64_t ld_up, const void* w_down, int64_t ld_down, uint32_t M, uint32_t D, uint32_t F,
                              uint32_t O, int dtype, int activation, void* dx, int64_t lddx, void* dw_gate, void* dw_up, void* dw_down,
                              void* workspace, uint64_t workspace_bytes, envidr_stream_t stream) {
    if (int rc = gated_checks("gated_mlp_backward", M, D, F, O, dtype, activation)) return rc;
    hipStream_t s = as_stream(stream);
    if (M == 0) {                                    // no rows: the weights' gradients are zero
        void* out[3] = {dw_gate, dw_up, dw_down};
        for (int i = 0; i < 3; ++i) {
            if (!out[i]) continue;
            const uint64_t n = (uint64_t)F * (i < 2 ? D : O) * (dtype_size(dtype) / 2u);
            const uint64_t blocks = (n + kBlock - 1) / kBlock, most = 16 * kCus;
            hipLaunchKernelGGL(k_zero, dim3((uint32_t)(blocks < most ? blocks : most)), dim3(kBlock), 0, s, static_cast<uint16_t*>(out[i]), n);
            if (int rc = check_launch("k_zero")) return rc;
        }
        return ENVIDR_OK;
    }
    ENVIDR_REQUIRE(dy && x && w_gate && w_up && w_down, "gated_mlp_backward: null pointer");
    const int64_t most = 1ll << 21;
    ENVIDR_REQUIRE(lddy >= 0 && ldx >= 0 && ld_gate >= 0 && ld_up >= 0 && ld_down >= 0 && lddy <= most && ldx <= most && ld_gate <= most && ld_up <= most && ld_down <= most,
                   "gated_mlp_backward: a row pitch is negative or above 2^21");
    ENVIDR_REQUIRE(!dx || (lddx >= D && lddx <= most), "gated_mlp_backward: lddx=%lld < D=%u, or above 2^21", (long long)lddx, D);
    if (int rc = workspace_checks("gated_mlp_backward", workspace, workspace_bytes, envidr_gated_mlp_workspace_bytes(M, D, F, O, dtype, 1))) return rc;
    const Weights w{w_gate, w_up, w_down, ld_gate, ld_up, ld_down};
    ENVIDR_FOR_DTYPE(dtype, E, return backward<E>(dy, lddy, x, ldx, w, M, D, F, O, dtype, activation, dx, lddx, dw_gate, dw_up, dw_down,
                                                  static_cast<char*>(workspace), s));
}

}  // extern "C"
