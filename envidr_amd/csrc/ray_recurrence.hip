// A gated linear recurrence along the samples of packed rays, forward and backward:
//   a_t = sigmoid(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) v_t  (blend)  or  a_t h_{t-1} + v_t,   every channel by itself
//   backward, from a ray's last sample to its first, E = d(last):  G_t = dh_t + E;  dv_t = (1 - a_t) G_t (or G_t);
//   dgate_t = G_t (h_{t-1} - v_t) a_t (1 - a_t)  (or G_t h_{t-1} a_t (1 - a_t));  E = a_t G_t.   dstate = E at the end.
// Bound: memory (3 streams forward, 5 backward).
//
// Decomposition.  Rays are of any length (one sample to all of them), so a ray is cut where the packed row index is a multiple of `piece`:
// a HEAD piece from its first row to the first such border, then one piece per border inside it.  A border lies inside at most one ray, so
// heads (N) and border pieces (T / piece) have fixed places and need no list and no count on the host: owner[k] is the ray that border k
// cuts, written by the ray itself.  Nothing is cleared beforehand: a place no ray wrote holds some old number, and a number is believed only
// if the ray of that number does contain the border.
//   k_scan_map     per ray: its borders' owner[], mark[] (the ray's number) on the rows of its head piece, named[] at its id
//   k_scan_sums    per border: the piece before it (backward: behind it) as the affine map  out = A in + B  it applies to the carried state
//   k_scan_join, k_scan_carry   the maps in order -> the state at every border
//   k_scan_forward / k_scan_backward   per piece: rows in blocks of kRows, the next block loaded under the present one; rows that neither a
//                  mark nor an owner claims get zeros, and ids that no ray names keep their state
// A ray that no border falls into is one piece and pays for none of the middle; of a cut one, whatever its length, the rows between a border and the
// next are read a second time by k_scan_sums (4096 rays of 36 rows on average: 43 % of the rays, half the rows).  With at most a row a ray or few rows
// in all nothing is cut: two launches instead of five.
// Lanes are channels, two each in the 16-bit types where C is even (a row of 128 channels is then one 256-byte access of a wave, not two of 128:
// 230 us a training pass of three sequences, 300 k rows, bf16; 233 with one channel a lane).  From 64 lanes a row on a wave has one piece, and rows,
// bounds and addresses live on the scalar unit; with fewer channels 64 / lanes pieces share a wave.
// The backward pass needs h_{t-1}.  It does not read the stored (rounded) h: the forward pass leaves the 32-bit state at every kRows-th row
// (`saved`), and a block's states are formed again from there in registers.
#include "blocks_common.hip.h"

#include <type_traits>

namespace envidr {
namespace {

constexpr uint32_t kRows = 8;           // rows of a block: what a lane holds in registers at once
constexpr uint32_t kCarryThreads = 1024, kCarryLanes = 16, kJoin = 64;         // 64 borders by 16 channels

struct ScanPlan {
    uint32_t piece;         // rows between borders, 0: nothing is cut
    uint32_t borders;       // T / piece rounded up (border 0 is never used)
    uint64_t states;        // saved states: one row of C for every kRows rows
};

ScanPlan scan_plan(uint64_t T, uint32_t N) {
    ScanPlan p{};
    // Not cut: at most 256 rows (46 us a training pass against 56 cut; at 512 rows 82 against 57), or at most a row a ray on average -- the step of
    // many rays with their states (1000 rays of one row, 64 channels: 16 us a training pass against 30 cut).  The price of the second: where most
    // rays are empty, a long one among them is walked by one wave (4096 rows in four rays, training: rays of 300 rows 90 us against 64 cut, of
    // 1000 rows 277 against 65).  Anything else may hide a ray that is nearly all of T.
    if (T > 256 && T > N) {
        // 64 rows, doubled until at most 8192 borders (128 segments) are left.  (Three sequences, 300 k rows of 128 channels in bf16: with
        // pieces of 256 rows and blocks of 16 a wave a SIMD is left to its own latencies -- sums 47, forward 51, backward 125 us; 34, 44, 73 so.)
        p.piece = 64;
        while ((T + p.piece - 1) / p.piece > 8192) p.piece *= 2;
        p.borders = (uint32_t)((T + p.piece - 1) / p.piece);
    }
    p.states = (T + kRows - 1) / kRows;
    return p;
}

struct Lanes {
    uint32_t lanes, groups;         // lanes a piece takes in a wave (a power of two), channel groups (grid.y)
};
Lanes lanes_of(uint32_t C, uint32_t V) {
    const uint32_t units = ceil_div(C, V);
    Lanes l{1, 0};
    while (l.lanes < 64u && l.lanes < units) l.lanes *= 2u;
    l.groups = ceil_div(units, l.lanes);
    return l;
}

struct ScanArgs {
    const void *gate, *value, *dh;
    const int32_t* rays;
    const float *state, *dlast;
    void *out0, *out1;              // h | dgate, dvalue
    float* last;                    // last | dstate
    float *sum_a, *sum_b;           // [borders][C]
    float *segment_a, *segment_b, *segment_in;      // [borders / kJoin][C]
    float* saved;                   // [states][C] or NULL
    int32_t *mark, *owner, *named;  // [T], [borders], [N]
    uint32_t T, N, C, piece, borders, lanes, piece_blocks, zero_blocks;
};

struct RayRows {
    uint32_t begin, end;    // begin == end: no rows
    int32_t id;
};

__device__ __forceinline__ RayRows ray_rows(const ScanArgs& a, uint32_t n) {
    const int32_t id = a.rays[3 * (size_t)n], off = a.rays[3 * (size_t)n + 1], cnt = a.rays[3 * (size_t)n + 2];
    const bool ok = cnt > 0 && off >= 0 && (uint64_t)(uint32_t)off + (uint32_t)cnt <= a.T;
    RayRows r;
    r.begin = ok ? (uint32_t)off : 0u;
    r.end = ok ? (uint32_t)off + (uint32_t)cnt : 0u;
    r.id = id >= 0 && (uint32_t)id < a.N ? id : -1;
    return r;
}

// the ray that border k cuts (its row k * piece is a row of it, and not the first): -1 if none
__device__ __forceinline__ int32_t border_owner(const ScanArgs& a, uint32_t k, RayRows& r) {
    if (k == 0 || k >= a.borders) return -1;
    const int32_t n = a.owner[k];
    if (n < 0 || (uint32_t)n >= a.N) return -1;
    r = ray_rows(a, (uint32_t)n);
    const uint32_t row = k * a.piece;
    return r.begin < row && row < r.end ? n : -1;
}

__device__ __forceinline__ uint32_t head_end(const ScanArgs& a, const RayRows& r) {
    return a.piece && r.end > r.begin ? min(r.end, (r.begin / a.piece + 1u) * a.piece) : r.end;
}

__global__ void __launch_bounds__(kBlock) k_scan_map(ScanArgs a) {
    const uint32_t n = blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63u;
    if (n >= a.N) return;
    const RayRows r = ray_rows(a, n);
    if (lane == 0 && r.id >= 0) a.named[r.id] = (int32_t)n;
    if (r.begin == r.end) return;
    for (uint32_t row = r.begin + lane; row < head_end(a, r); row += 64u) a.mark[row] = (int32_t)n;
    if (a.piece)
        for (uint32_t k = r.begin / a.piece + 1u + lane; k <= (r.end - 1u) / a.piece; k += 64u) a.owner[k] = (int32_t)n;
}

// UNI: a wave has one piece, so what depends on the piece is the same for all lanes
template <bool UNI> __device__ __forceinline__ uint32_t same(uint32_t v) { return UNI ? (uint32_t)__builtin_amdgcn_readfirstlane((int)v) : v; }

// the kRows rows from row `first` on; rows outside [begin, end) repeat the nearest row inside
template <class E, int V> struct Block {
    Pack<E, V> r[kRows];
    __device__ __forceinline__ void load(const void* base, uint32_t first, uint32_t begin, uint32_t end, uint32_t C, uint32_t c) {
#pragma unroll
        for (uint32_t j = 0; j < kRows; ++j) r[j] = load_pack<E, V>(static_cast<const E*>(base) + (uint64_t)min(max(first + j, begin), end - 1u) * C + c);
    }
    __device__ __forceinline__ float at(uint32_t j, int i) const { return to_f32(r[j].v[i]); }
};
template <class E, int V> __device__ __forceinline__ void store_row(void* base, uint32_t row, uint32_t C, uint32_t c, const float (&v)[V]) {
    Pack<E, V> p;
#pragma unroll
    for (int i = 0; i < V; ++i) p.v[i] = from_f32<E>(v[i]);
    store_pack(static_cast<E*>(base) + (uint64_t)row * C + c, p);
}

// where a lane works: the piece's rows, its ray, its channels.  false: nothing to do
struct Place {
    RayRows ray;
    uint32_t begin, end, c;
    bool is_head;
};
template <int V, bool UNI> __device__ __forceinline__ bool find_place(const ScanArgs& a, Place& p) {
    const uint32_t lanes = UNI ? 64u : a.lanes, slot = same<UNI>(blockIdx.x * (kBlock / lanes) + threadIdx.x / lanes);
    p.c = (blockIdx.y * lanes + (threadIdx.x & (lanes - 1u))) * V;
    if (p.c >= a.C) return false;
    if (slot < a.N) {
        p.ray = ray_rows(a, slot);
        p.is_head = true;
        p.begin = p.ray.begin;
        p.end = head_end(a, p.ray);
        return true;
    }
    const uint32_t k = slot - a.N;
    if (border_owner(a, k, p.ray) < 0) return false;
    p.is_head = false;
    p.begin = k * a.piece;
    p.end = min(p.ray.end, p.begin + a.piece);
    return true;
}

// The blocks behind the pieces'.  Rows that no ray claims get zeros (64 rows a wave); ids that no ray names: to[id] = from[id], or zeros.
template <class E> __device__ __forceinline__ void fill_rest(const ScanArgs& a, void* out0, void* out1, const float* from, float* to) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t block = blockIdx.x - a.piece_blocks;
    if (block >= a.zero_blocks) {
        block -= a.zero_blocks;
        const uint32_t first = (block * (kBlock / 64) + (threadIdx.x >> 6)) * 64u, id = first + lane;
        bool is_named = true;
        if (id < a.N) {
            const int32_t n = a.named[id];
            is_named = n >= 0 && (uint32_t)n < a.N && a.rays[3 * (size_t)(uint32_t)n] == (int32_t)id;
        }
        uint64_t left = __ballot(!is_named);
        while (left && to) {
            const uint32_t j = (uint32_t)__builtin_ctzll(left);
            left &= left - 1;
            for (uint32_t c = lane; c < a.C; c += 64u) to[(uint64_t)(first + j) * a.C + c] = from ? from[(uint64_t)(first + j) * a.C + c] : 0.0f;
        }
        return;
    }
    const uint32_t first = (block * (kBlock / 64) + (threadIdx.x >> 6)) * 64u, row = first + lane;
    bool claimed = true;
    if (row < a.T) {
        const int32_t n = a.mark[row];
        claimed = false;
        if (n >= 0 && (uint32_t)n < a.N) {
            const RayRows r = ray_rows(a, (uint32_t)n);
            claimed = r.begin <= row && row < r.end;
        }
        if (!claimed && a.piece) {
            RayRows r;
            claimed = border_owner(a, row / a.piece, r) >= 0 && row < r.end;
        }
    }
    uint64_t left = __ballot(!claimed);
    while (left) {
        const uint32_t j = (uint32_t)__builtin_ctzll(left);
        left &= left - 1;
        const uint64_t at = (uint64_t)(first + j) * a.C;
        for (uint32_t c = lane; c < a.C; c += 64u) {
            static_cast<E*>(out0)[at + c] = from_f32<E>(0.0f);
            if (out1) static_cast<E*>(out1)[at + c] = from_f32<E>(0.0f);
        }
    }
}

template <int V> __device__ __forceinline__ void load_f32(const float* p, uint64_t at, float (&h)[V]) {
    const Pack<float, V> x = load_pack<float, V>(p + at);
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = x.v[i];
}
template <int V> __device__ __forceinline__ void store_f32(float* p, uint64_t at, const float (&h)[V]) {
    Pack<float, V> x;
#pragma unroll
    for (int i = 0; i < V; ++i) x.v[i] = h[i];
    store_pack(p + at, x);
}
template <int V> __device__ __forceinline__ void load_state(const float* s, int32_t id, uint32_t C, uint32_t c, float (&h)[V]) {
    if (s && id >= 0) {
        load_f32<V>(s, (uint64_t)(uint32_t)id * C + c, h);
        return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = 0.0f;
}

// One step.  Blend: a h + (1 - a) v, formed as (1 - w) near + w far with w the smaller weight and `near` what it leaves most of: an open gate (a
// near 1, whose rounding would be all of 1 - a) goes by 1 - a, a closed one by a, and every rounding is one of a |h| or (1 - a) |v|.  (As
// h + (1 - a) (v - h) a closed gate would leave 2^-24 of the h that it replaces.)  near's own infinity must not meet itself: w times the largest number
// taken from it leaves it.
template <bool BLEND> __device__ __forceinline__ float step(float gate, float h, float a, float an, float v) {
    if constexpr (!BLEND) return fmaf(a, h, v);
    const bool closed = gate < 0.0f;
    const float w = closed ? a : an, near = closed ? v : h, far = closed ? h : v;
    return fmaf(w, far, fmaf(-w, __builtin_amdgcn_fmed3f(near, -3.402823466e38f, 3.402823466e38f), near));
}

// Affine maps in order: first, then second.  A map that forgets its input -- a border of nobody, or the first border of a ray, which has the ray's
// own initial state in B -- is marked by A = -0: what is carried there may be another ray's NaN or infinity.  (A product of sigmoids that got too
// small is +0 and forgets nothing: a NaN stays one along its own ray.)  The mark outlives a product with a later positive A.
constexpr float kForget = -0.0f;
__device__ __forceinline__ bool forgets(float A) { return __builtin_bit_cast(uint32_t, A) == 0x80000000u; }
// That +0 is a number above zero, and an infinity times it is one.
__device__ __forceinline__ float apply(float A, float B, float in) {
    if (forgets(A)) return B;
    return A == 0.0f && __builtin_isinf(in) ? in + B : fmaf(A, in, B);
}

// the state that crosses border k (forward: h before its row; backward: E behind the row before it)
template <int V> __device__ __forceinline__ void load_carry(const ScanArgs& a, uint32_t k, uint32_t c, float (&h)[V]) {
    const uint64_t at = (uint64_t)k * a.C + c, seg = (uint64_t)(k / kJoin) * a.C + c;
    float A[V], in[V];
    load_f32<V>(a.sum_a, at, A);
    load_f32<V>(a.sum_b, at, h);
    load_f32<V>(a.segment_in, seg, in);
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = apply(A[i], h[i], in[i]);
}

template <class E, int V, bool BLEND, bool UNI> __global__ void __launch_bounds__(kBlock) k_scan_forward(ScanArgs a) {
    if (blockIdx.x >= a.piece_blocks) {
        if (blockIdx.y == 0) fill_rest<E>(a, a.out0, nullptr, a.state, a.last);
        return;
    }
    Place p;
    if (!find_place<V, UNI>(a, p)) return;
    float h[V];
    if (p.is_head) load_state<V>(a.state, p.ray.id, a.C, p.c, h);
    else load_carry<V>(a, p.begin / a.piece, p.c, h);
    if (p.begin < p.end) {
        struct Rows {
            Block<E, V> g, v;
        } now, next;
        auto fetch = [&](Rows& x, uint32_t first) {
            x.g.load(a.gate, first, p.begin, p.end, a.C, p.c);
            x.v.load(a.value, first, p.begin, p.end, a.C, p.c);
        };
        auto work = [&](const Rows& x, uint32_t first) {
            if (a.saved && first > p.ray.begin) store_f32<V>(a.saved, (uint64_t)(first / kRows) * a.C + p.c, h);
#pragma unroll
            for (uint32_t j = 0; j < kRows; ++j) {
                const uint32_t row = first + j;
                if (row < p.begin || row >= p.end) continue;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float s, sn;
                    sigmoid_pair<sizeof(E) == 4>(x.g.at(j, i), s, sn);
                    h[i] = step<BLEND>(x.g.at(j, i), h[i], s, sn, x.v.at(j, i));
                }
                store_row<E, V>(a.out0, row, a.C, p.c, h);
            }
        };
        uint32_t first = p.begin / kRows * kRows;
        fetch(now, first);
        for (;;) {
            if (first + kRows < p.end) fetch(next, first + kRows);
            work(now, first);
            if ((first += kRows) >= p.end) break;
            if (first + kRows < p.end) fetch(now, first + kRows);
            work(next, first);
            if ((first += kRows) >= p.end) break;
        }
    }
    if (p.end == p.ray.end && p.ray.id >= 0) store_f32<V>(a.last, (uint64_t)(uint32_t)p.ray.id * a.C + p.c, h);
}

template <class E, int V, bool BLEND, bool UNI> __global__ void __launch_bounds__(kBlock) k_scan_backward(ScanArgs a) {
    if (blockIdx.x >= a.piece_blocks) {
        if (blockIdx.y == 0) fill_rest<E>(a, a.out0, a.out1, a.dlast, a.last);
        return;
    }
    Place p;
    if (!find_place<V, UNI>(a, p)) return;
    float e[V];
    if (p.end == p.ray.end) load_state<V>(a.dlast, p.ray.id, a.C, p.c, e);
    else load_carry<V>(a, p.end / a.piece, p.c, e);
    if (p.begin < p.end) {
        struct Rows {
            Block<E, V> g, v, d;
            float h[V];
        } now, next;
        const uint32_t first0 = p.begin / kRows * kRows;
        auto fetch = [&](Rows& x, uint32_t first) {
            x.g.load(a.gate, first, p.begin, p.end, a.C, p.c);
            x.v.load(a.value, first, p.begin, p.end, a.C, p.c);
            x.d.load(a.dh, first, p.begin, p.end, a.C, p.c);
            if (first > p.ray.begin) load_f32<V>(a.saved, (uint64_t)(first / kRows) * a.C + p.c, x.h);
            else load_state<V>(a.state, p.ray.id, a.C, p.c, x.h);
        };
        auto work = [&](Rows& x, uint32_t first) {
            float before[kRows][V];
#pragma unroll
            for (uint32_t j = 0; j < kRows; ++j) {
                const uint32_t row = first + j;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    before[j][i] = x.h[i];
                    float s, sn;
                    sigmoid_pair<sizeof(E) == 4>(x.g.at(j, i), s, sn);
                    const float then = step<BLEND>(x.g.at(j, i), x.h[i], s, sn, x.v.at(j, i));
                    x.h[i] = row >= p.begin ? then : x.h[i];
                }
            }
#pragma unroll
            for (uint32_t jj = 0; jj < kRows; ++jj) {
                const uint32_t j = kRows - 1u - jj, row = first + j;
                if (row < p.begin || row >= p.end) continue;
                float dg[V], dv[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    // (formed again: kept from the pass above, the pairs would take 32 V registers more and halve the waves in flight)
                    float s, sn, gate = x.g.at(j, i);
                    asm("" : "+v"(gate));
                    sigmoid_pair<sizeof(E) == 4>(gate, s, sn);
                    const float G = x.d.at(j, i) + e[i], from = BLEND ? before[j][i] - x.v.at(j, i) : before[j][i];
                    dv[i] = BLEND ? G * sn : G;
                    e[i] = s * G;
                    dg[i] = e[i] * sn * from;
                }
                store_row<E, V>(a.out0, row, a.C, p.c, dg);
                store_row<E, V>(a.out1, row, a.C, p.c, dv);
            }
        };
        uint32_t first = (p.end - 1u) / kRows * kRows;
        fetch(now, first);
        for (;;) {
            if (first > first0) fetch(next, first - kRows);
            work(now, first);
            if (first == first0) break;
            first -= kRows;
            if (first > first0) fetch(now, first - kRows);
            work(next, first);
            if (first == first0) break;
            first -= kRows;
        }
    }
    if (p.is_head && a.last && p.ray.id >= 0) store_f32<V>(a.last, (uint64_t)(uint32_t)p.ray.id * a.C + p.c, e);
}

// the affine map of the piece before border k (forward: what it does to h) or behind it (backward: what it does to E)
template <class E, int V, bool BLEND, bool BACK, bool UNI> __global__ void __launch_bounds__(kBlock) k_scan_sums(ScanArgs a) {
    const uint32_t lanes = UNI ? 64u : a.lanes, k = same<UNI>(blockIdx.x * (kBlock / lanes) + threadIdx.x / lanes);
    const uint32_t c = (blockIdx.y * lanes + (threadIdx.x & (lanes - 1u))) * V;
    RayRows ray;
    if (c >= a.C || border_owner(a, k, ray) < 0) return;
    const uint32_t begin = BACK ? k * a.piece : max(ray.begin, (k - 1u) * a.piece), end = BACK ? min(ray.end, (k + 1u) * a.piece) : k * a.piece;
    float A[V], B[V];
#pragma unroll
    for (int i = 0; i < V; ++i) { A[i] = 1.0f; B[i] = 0.0f; }
    const uint32_t first0 = begin / kRows * kRows, last0 = (end - 1u) / kRows * kRows;
    struct Rows {
        Block<E, V> g, v;
    } now, next;
    auto fetch = [&](Rows& x, uint32_t first) {
        x.g.load(a.gate, first, begin, end, a.C, c);
        x.v.load(BACK ? a.dh : a.value, first, begin, end, a.C, c);
    };
    auto work = [&](const Rows& x, uint32_t first) {
#pragma unroll
        for (uint32_t jj = 0; jj < kRows; ++jj) {
            const uint32_t j = BACK ? kRows - 1u - jj : jj, row = first + j;
            if (row < begin || row >= end) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float s, sn;
                sigmoid_pair<sizeof(E) == 4>(x.g.at(j, i), s, sn);
                const float y = x.v.at(j, i);
                B[i] = BACK ? s * (B[i] + y) : step<BLEND>(x.g.at(j, i), B[i], s, sn, y);
                A[i] *= s;
            }
        }
    };
    uint32_t first = BACK ? last0 : first0;
    const uint32_t stop = BACK ? first0 : last0;
    auto then = [&](uint32_t f) { return BACK ? f - kRows : f + kRows; };
    fetch(now, first);
    for (;;) {
        if (first != stop) fetch(next, then(first));
        work(now, first);
        if (first == stop) break;
        first = then(first);
        if (first != stop) fetch(now, then(first));
        work(next, first);
        if (first == stop) break;
        first = then(first);
    }
    store_f32<V>(a.sum_a, (uint64_t)k * a.C + c, A);
    store_f32<V>(a.sum_b, (uint64_t)k * a.C + c, B);
}

// The maps at `mine` of kJoin x `lanes` threads, run r's after those of the runs before it: an inclusive scan over the runs (of 0 .. kJoin - 1).
// Ends with a barrier behind the last read of s_a, s_b.
__device__ __forceinline__ void join_runs(float* s_a, float* s_b, uint32_t run, uint32_t runs, uint32_t lanes, float& A, float& B) {
    for (uint32_t span = 1; span < runs; span *= 2) {
        s_a[threadIdx.x] = A;
        s_b[threadIdx.x] = B;
        __syncthreads();
        if (run >= span) {
            B = apply(A, B, s_b[threadIdx.x - span * lanes]);
            A = forgets(A) ? A : A * s_a[threadIdx.x - span * lanes];
        }
        __syncthreads();
    }
}

// Two kernels join the maps of all borders in order (backward: in reverse), whatever ray they belong to -- a ray's first border forgets what was
// before it.  k_scan_join: within segments of kJoin borders, each border's map becomes the one from its segment's start; k_scan_carry: the
// segments' own maps -> what enters each segment.  The state at a border is then sum_a * segment_in + sum_b.
// (One workgroup a cut ray, walking its borders in 64 runs, took 41 us for 2900 borders: memory's latency a batch of loads.)
template <bool BACK> __global__ void __launch_bounds__(kCarryThreads) k_scan_join(ScanArgs a) {
    __shared__ float s_a[kCarryThreads], s_b[kCarryThreads];
    const uint32_t lane = threadIdx.x & (a.lanes - 1u), run = threadIdx.x / a.lanes, runs = kCarryThreads / a.lanes, c = blockIdx.y * a.lanes + lane;
    // (with fewer than sixteen channels there are more runs than a segment has borders: the rest idle)
    const uint32_t k = blockIdx.x * kJoin + (BACK ? kJoin - 1u - run : run);
    const bool on = run < kJoin && c < a.C && k < a.borders;
    RayRows ray;
    float A = kForget, B = 0.0f;
    if (on && border_owner(a, k, ray) >= 0) {
        const uint64_t at = (uint64_t)k * a.C + c;
        A = a.sum_a[at];
        B = a.sum_b[at];
        if (k == (BACK ? (ray.end - 1u) / a.piece : ray.begin / a.piece + 1u)) {
            const float* start = BACK ? a.dlast : a.state;
            B = apply(A, B, start && ray.id >= 0 ? start[(uint64_t)(uint32_t)ray.id * a.C + c] : 0.0f);
            A = kForget;
        }
    }
    join_runs(s_a, s_b, run, runs, a.lanes, A, B);
    if (on) {
        const uint64_t at = (uint64_t)k * a.C + c;
        a.sum_a[at] = A;
        a.sum_b[at] = B;
    }
    // (the segment's own map: its last border's in the order; the missing borders of the last segment come first backward, and forget)
    if (c < a.C && run == kJoin - 1u) {
        const uint64_t at = (uint64_t)blockIdx.x * a.C + c;
        a.segment_a[at] = A;
        a.segment_b[at] = B;
    }
}

template <bool BACK> __global__ void __launch_bounds__(kCarryThreads) k_scan_carry(ScanArgs a) {
    __shared__ float s_a[kCarryThreads], s_b[kCarryThreads];
    const uint32_t lane = threadIdx.x & (a.lanes - 1u), run = threadIdx.x / a.lanes, runs = kCarryThreads / a.lanes, c = blockIdx.x * a.lanes + lane;
    const uint32_t segments = (a.borders + kJoin - 1u) / kJoin;
    const bool on = c < a.C;
    float in = 0.0f;                                 // what enters the first segment of this round of `runs` segments
    for (uint32_t s0 = 0; s0 < segments; s0 += runs) {
        const uint32_t s = s0 + run, g = BACK ? segments - 1u - s : s;
        const bool mine = on && s < segments;
        float A = kForget, B = 0.0f;
        if (mine) {
            A = a.segment_a[(uint64_t)g * a.C + c];
            B = a.segment_b[(uint64_t)g * a.C + c];
        }
        join_runs(s_a, s_b, run, runs, a.lanes, A, B);
        s_a[threadIdx.x] = apply(A, B, in);          // what leaves segment s
        __syncthreads();
        if (mine) a.segment_in[(uint64_t)g * a.C + c] = run ? s_a[threadIdx.x - a.lanes] : in;
        in = s_a[(runs - 1u) * a.lanes + lane];
        __syncthreads();
    }
}

// the places of the workspace: the borders' and segments' maps, then marks, owners and names when they are not kept in `saved`
uint64_t table_words(const ScanPlan& p, uint64_t T, uint32_t N) { return round_up64(T, 4) + round_up64(p.borders, 4) + round_up64(N, 4); }
uint64_t sum_words(const ScanPlan& p, uint32_t C) { return round_up64((uint64_t)p.borders * C, 4); }
uint64_t segment_words(const ScanPlan& p, uint32_t C) { return round_up64((uint64_t)ceil_div(p.borders, kJoin) * C, 4); }
uint64_t sums_words(const ScanPlan& p, uint32_t C) { return 2ull * sum_words(p, C) + 3ull * segment_words(p, C); }

template <class E, int V, bool BACK, bool BLEND, bool UNI> int launch_scan(const ScanArgs& a, const ScanPlan& p, const Lanes& l, hipStream_t s) {
    const uint32_t per_block = kBlock / l.lanes;
    if (!BACK && a.N > 0) {
        hipLaunchKernelGGL(k_scan_map, dim3(ceil_div(a.N, kBlock / 64u)), dim3(kBlock), 0, s, a);
        if (int rc = check_launch("k_scan_map")) return rc;
    }
    if (p.piece) {
        hipLaunchKernelGGL((k_scan_sums<E, V, BLEND, BACK, UNI>), dim3(ceil_div(p.borders, per_block), l.groups), dim3(kBlock), 0, s, a);
        if (int rc = check_launch("k_scan_sums")) return rc;
        ScanArgs b = a;
        b.lanes = l.lanes < kCarryLanes ? l.lanes : kCarryLanes;
        hipLaunchKernelGGL((k_scan_join<BACK>), dim3(ceil_div(p.borders, kJoin), ceil_div(a.C, b.lanes)), dim3(kCarryThreads), 0, s, b);
        if (int rc = check_launch("k_scan_join")) return rc;
        hipLaunchKernelGGL((k_scan_carry<BACK>), dim3(ceil_div(a.C, b.lanes)), dim3(kCarryThreads), 0, s, b);
        if (int rc = check_launch("k_scan_carry")) return rc;
    }
    const dim3 grid(a.piece_blocks + a.zero_blocks + ceil_div(a.N, kBlock), l.groups);
    if constexpr (BACK) hipLaunchKernelGGL((k_scan_backward<E, V, BLEND, UNI>), grid, dim3(kBlock), 0, s, a);
    else hipLaunchKernelGGL((k_scan_forward<E, V, BLEND, UNI>), grid, dim3(kBlock), 0, s, a);
    return check_launch(BACK ? "k_scan_backward" : "k_scan_forward");
}

template <class E, bool BACK> int run_scan(ScanArgs a, bool blend, void* workspace, float* saved, hipStream_t s) {
    const ScanPlan p = scan_plan(a.T, a.N);
    float* w = static_cast<float*>(workspace);
    a.sum_a = w;
    a.sum_b = a.sum_a + sum_words(p, a.C);
    a.segment_a = a.sum_b + sum_words(p, a.C);
    a.segment_b = a.segment_a + segment_words(p, a.C);
    a.segment_in = a.segment_b + segment_words(p, a.C);
    float* tables = saved ? saved + round_up64(p.states * a.C, 4) : a.segment_in + segment_words(p, a.C);
    a.mark = reinterpret_cast<int32_t*>(tables);
    a.owner = a.mark + round_up64(a.T, 4);
    a.named = a.owner + round_up64(p.borders, 4);
    a.saved = saved;
    a.piece = p.piece;
    a.borders = p.borders;
    const bool pairs = sizeof(E) == 2 && a.C % 2 == 0;
    const Lanes l = lanes_of(a.C, pairs ? 2 : 1);
    a.lanes = l.lanes;
    const uint64_t slots = (uint64_t)a.N + p.borders, per_block = kBlock / l.lanes;
    a.piece_blocks = (uint32_t)((slots + per_block - 1) / per_block);
    a.zero_blocks = ceil_div(a.T, kBlock);          // (64 rows a wave)
    auto go = [&](auto v, auto b) {
        constexpr int V = decltype(v)::value;
        constexpr bool BLEND = decltype(b)::value;
        return l.lanes == 64 ? launch_scan<E, V, BACK, BLEND, true>(a, p, l, s) : launch_scan<E, V, BACK, BLEND, false>(a, p, l, s);
    };
    if constexpr (sizeof(E) == 2)
        if (pairs) return blend ? go(std::integral_constant<int, 2>{}, std::true_type{}) : go(std::integral_constant<int, 2>{}, std::false_type{});
    return blend ? go(std::integral_constant<int, 1>{}, std::true_type{}) : go(std::integral_constant<int, 1>{}, std::false_type{});
}

// a launch holds fewer than 2^32 threads: k_scan_map takes 64 a ray; the passes at most 64 a piece (a head of every ray, 8192 border pieces), one a
// row and one an id
bool scan_fits(uint64_t T, uint32_t N, uint32_t C) { return T <= 0x7FFFFFFFull && 64ull * (N + 8192ull + 8u) + T + N < 1ull << 32 && C <= (1u << 19); }

int scan_checks(const char* what, uint64_t T, uint32_t N, uint32_t C, int dtype, const void* workspace, uint64_t workspace_bytes) {
    ENVIDR_REQUIRE(dtype_ok(dtype), "%s: unknown dtype %d", what, dtype);
    ENVIDR_REQUIRE(C >= 1, "%s: no channels", what);
    ENVIDR_REQUIRE(scan_fits(T, N, C), "%s: T=%llu, N=%u or C=%u is too large", what, (unsigned long long)T, N, C);
    ENVIDR_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= envidr_ray_recurrence_workspace_bytes(T, N, C) && (workspace || (T == 0 && N == 0)),
                   "%s: workspace of %llu bytes, %llu needed", what, (unsigned long long)workspace_bytes, (unsigned long long)envidr_ray_recurrence_workspace_bytes(T, N, C));
    return ENVIDR_OK;
}

}  // namespace
}  // namespace envidr

using namespace envidr;

extern "C" {

uint64_t envidr_ray_recurrence_saved_floats(uint64_t T, uint32_t N, uint32_t C) {
    if (!scan_fits(T, N, C)) return 0;
    const ScanPlan p = scan_plan(T, N);
    return round_up64(p.states * C, 4) + table_words(p, T, N);
}

uint64_t envidr_ray_recurrence_workspace_bytes(uint64_t T, uint32_t N, uint32_t C) {
    if (!scan_fits(T, N, C)) return 0;
    const ScanPlan p = scan_plan(T, N);
    return 4ull * (sums_words(p, C) + table_words(p, T, N));
}

int envidr_ray_recurrence_forward(const void* gate, const void* value, const int32_t* rays, const float* state, uint64_t T, uint32_t N,
                                  uint32_t C, int dtype, int blend, void* h, float* last, float* saved, void* workspace,
                                  uint64_t workspace_bytes, envidr_stream_t stream) {
    if (int rc = scan_checks("ray_recurrence_forward", T, N, C, dtype, workspace, workspace_bytes)) return rc;
    if (N == 0 && T == 0) return ENVIDR_OK;
    ENVIDR_REQUIRE((gate && value && h) || T == 0, "ray_recurrence_forward: null pointer");
    ENVIDR_REQUIRE((rays && last) || N == 0, "ray_recurrence_forward: null pointer");
    ScanArgs a{};
    a.gate = gate; a.value = value; a.rays = rays; a.state = state; a.out0 = h; a.last = last;
    a.T = (uint32_t)T; a.N = N; a.C = C;
    ENVIDR_FOR_DTYPE(dtype, E, return (run_scan<E, false>(a, blend != 0, workspace, saved, as_stream(stream))));
}

int envidr_ray_recurrence_backward(const void* dh, const float* dlast, const void* gate, const void* value, const int32_t* rays,
                                   const float* state, const float* saved, uint64_t T, uint32_t N, uint32_t C, int dtype, int blend,
                                   void* dgate, void* dvalue, float* dstate, void* workspace, uint64_t workspace_bytes,
                                   envidr_stream_t stream) {
    if (int rc = scan_checks("ray_recurrence_backward", T, N, C, dtype, workspace, workspace_bytes)) return rc;
    if (N == 0 && T == 0) return ENVIDR_OK;
    ENVIDR_REQUIRE(((dh && gate && value && dgate && dvalue) || T == 0) && saved, "ray_recurrence_backward: null pointer");
    ENVIDR_REQUIRE(rays || N == 0, "ray_recurrence_backward: null pointer");
    ScanArgs a{};
    a.dh = dh; a.dlast = dlast; a.gate = gate; a.value = value; a.rays = rays; a.state = state; a.out0 = dgate; a.out1 = dvalue; a.last = dstate;
    a.T = (uint32_t)T; a.N = N; a.C = C;
    ENVIDR_FOR_DTYPE(dtype, E, return (run_scan<E, true>(a, blend != 0, workspace, const_cast<float*>(saved), as_stream(stream))));
}

}  // extern "C"
