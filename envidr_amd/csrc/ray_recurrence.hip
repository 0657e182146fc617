// A gated linear recurrence along the samples of packed rays, forward and backward:
//   a_t = sigmoid(gate_t),  h_t = a_t h_{t-1} + (1 - a_t) v_t  (blend)  or  a_t h_{t-1} + v_t,   every channel by itself
//   backward, from a ray's last sample to its first, E = d(last):  G_t = dh_t + E;  dv_t = (1 - a_t) G_t (or G_t);
//   dgate_t = G_t (h_{t-1} - v_t) a_t (1 - a_t)  (or G_t h_{t-1} a_t (1 - a_t));  E = a_t G_t.   dstate = E at the end.
// Bound: memory (3 streams forward, 5 backward).
//
// Decomposition.  Rays are of any length (one sample to all of them), so a ray is cut where the packed row index is a multiple of kPiece:
// a HEAD piece from its first row to the first such border, then one piece per border inside it.  A border lies inside at most one ray, so
// heads (N) and border pieces (T / kPiece) have fixed places and need no list and no count on the host: owner[k] is the ray that border k
// cuts, written by the ray itself.  Nothing is cleared beforehand: a place no ray wrote holds some old number, and a number is believed only
// if the ray of that number does contain the border.
//   k_scan_map     per ray: its borders' owner[], and mark[] (the ray's number) on the rows of its head piece
//   k_scan_sums    per border: the piece before it (backward: behind it) as the affine map  out = A in + B  it applies to the carried state
//   k_scan_carry   per cut ray: the maps in order -> the state at every border (sixteen waves take runs of borders, then one pass joins them)
//   k_scan_forward / k_scan_backward   per piece: rows in blocks of kRows; rows that neither a mark nor an owner claims get zeros
// Short rays are one piece each and pay for none of the middle; cut rays are read twice by k_scan_sums.  With few rows a ray (T <= 4 N) or
// few rows in all nothing is cut: two launches instead of four.
// Lanes are channels: 64 / (lanes a piece) pieces share a wave when there are fewer than 64 channels.
// The backward pass needs h_{t-1}.  It does not read the stored (rounded) h: the forward pass leaves the 32-bit state at every kRows-th row
// (`saved`), and a block's states are formed again from there in registers.
#include "blocks_common.hip.h"

namespace envidr {
namespace {

constexpr uint32_t kPiece = 256;        // rows between borders
constexpr uint32_t kRows = 16;          // rows of a block: what a lane holds in registers at once
constexpr uint32_t kCarryThreads = 1024;

struct ScanPlan {
    bool cut;               // rays are cut at borders
    uint32_t borders;       // T / kPiece rounded up (border 0 is never used), 0 when nothing is cut
    uint32_t lanes;         // lanes a piece takes in a wave (a power of two)
    uint32_t groups;        // channel groups (grid.y)
    uint64_t states;        // saved states: one row of C for every kRows rows
};

template <int V> ScanPlan scan_plan(uint64_t T, uint32_t N, uint32_t C) {
    ScanPlan p;
    p.cut = T > kPiece && T > 4ull * N;
    p.borders = p.cut ? (uint32_t)((T + kPiece - 1) / kPiece) : 0u;
    const uint32_t units = ceil_div(C, (uint32_t)V);
    p.lanes = 1;
    while (p.lanes < 64u && p.lanes < units) p.lanes *= 2u;
    p.groups = ceil_div(units, p.lanes);
    p.states = (T + kRows - 1) / kRows;
    return p;
}

struct ScanArgs {
    const void *gate, *value, *dh;
    const int32_t* rays;
    const float *state, *dlast;
    void *out0, *out1;              // h | dgate, dvalue
    float* last;                    // last | dstate
    float *sum_a, *sum_b, *carry;   // [borders][C]
    float* saved;                   // [states][C] or NULL
    int32_t *mark, *owner;          // [T], [borders]
    uint32_t T, N, C, borders, lanes, piece_blocks;
    bool cut;
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

// the ray that border k cuts (its row k * kPiece is a row of it, and not the first): -1 if none
__device__ __forceinline__ int32_t border_owner(const ScanArgs& a, uint32_t k, RayRows& r) {
    if (k == 0 || k >= a.borders) return -1;
    const int32_t n = a.owner[k];
    if (n < 0 || (uint32_t)n >= a.N) return -1;
    r = ray_rows(a, (uint32_t)n);
    const uint32_t row = k * kPiece;
    return r.begin < row && row < r.end ? n : -1;
}

__global__ void __launch_bounds__(kBlock) k_scan_map(ScanArgs a) {
    const uint32_t n = blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63u;
    if (n >= a.N) return;
    const RayRows r = ray_rows(a, n);
    if (r.begin == r.end) return;
    const uint32_t head = a.cut ? min(r.end, (r.begin / kPiece + 1u) * kPiece) : r.end;
    for (uint32_t row = r.begin + lane; row < head; row += 64u) a.mark[row] = (int32_t)n;
    if (a.cut)
        for (uint32_t k = r.begin / kPiece + 1u + lane; k <= (r.end - 1u) / kPiece; k += 64u) a.owner[k] = (int32_t)n;
}

// V channels of one row
template <class E, int V> __device__ __forceinline__ void load_row(const void* base, uint64_t at, float (&v)[V]) {
    const Pack<E, V> p = load_pack<E, V>(static_cast<const E*>(base) + at);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f32(p.v[i]);
}
template <class E, int V> __device__ __forceinline__ void store_row(void* base, uint64_t at, const float (&v)[V]) {
    Pack<E, V> p;
#pragma unroll
    for (int i = 0; i < V; ++i) p.v[i] = from_f32<E>(v[i]);
    store_pack(static_cast<E*>(base) + at, p);
}

// the kRows rows from row `first` on; rows outside [begin, end) repeat the nearest row inside
template <class E, int V> struct Block {
    Pack<E, V> r[kRows];
    __device__ __forceinline__ void load(const void* base, uint32_t first, uint32_t begin, uint32_t end, uint64_t C, uint32_t c) {
#pragma unroll
        for (uint32_t j = 0; j < kRows; ++j) {
            const uint32_t row = min(max(first + j, begin), end - 1u);
            r[j] = load_pack<E, V>(static_cast<const E*>(base) + (uint64_t)row * C + c);
        }
    }
};

// where a lane works: the piece's rows, its ray, its channels.  false: nothing to do
struct Place {
    RayRows ray;
    uint32_t begin, end, c;
    bool is_head;
};
template <int V> __device__ __forceinline__ bool find_place(const ScanArgs& a, Place& p) {
    const uint32_t per_block = kBlock / a.lanes, slot = blockIdx.x * per_block + threadIdx.x / a.lanes;
    p.c = (blockIdx.y * a.lanes + (threadIdx.x & (a.lanes - 1u))) * V;
    if (p.c >= a.C) return false;
    if (slot < a.N) {
        p.ray = ray_rows(a, slot);
        p.is_head = true;
        p.begin = p.ray.begin;
        p.end = a.cut && p.ray.end > p.ray.begin ? min(p.ray.end, (p.begin / kPiece + 1u) * kPiece) : p.ray.end;
        return true;
    }
    const uint32_t k = slot - a.N;
    if (border_owner(a, k, p.ray) < 0) return false;
    p.is_head = false;
    p.begin = k * kPiece;
    p.end = min(p.ray.end, p.begin + kPiece);
    return true;
}

// rows that no ray claims get zeros: the blocks behind the pieces' take 64 rows a wave
template <class E> __device__ __forceinline__ void zero_unclaimed(const ScanArgs& a, void* out0, void* out1) {
    const uint32_t lane = threadIdx.x & 63u, first = ((blockIdx.x - a.piece_blocks) * (kBlock / 64) + (threadIdx.x >> 6)) * 64u, row = first + lane;
    bool claimed = true;
    if (row < a.T) {
        const int32_t n = a.mark[row];
        claimed = false;
        if (n >= 0 && (uint32_t)n < a.N) {
            const RayRows r = ray_rows(a, (uint32_t)n);
            claimed = r.begin <= row && row < r.end;
        }
        if (!claimed && a.cut) {
            RayRows r;
            claimed = border_owner(a, row / kPiece, r) >= 0 && row < r.end;
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

template <int V> __device__ __forceinline__ void load_state(const float* s, int32_t id, uint32_t C, uint32_t c, float (&h)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) h[i] = s && id >= 0 ? s[(uint64_t)(uint32_t)id * C + c + i] : 0.0f;
}
template <int V> __device__ __forceinline__ void store_f32(float* p, uint64_t at, const float (&h)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) p[at + i] = h[i];
}

template <bool BLEND> __device__ __forceinline__ float step(float h, float a, float an, float v) {
    return BLEND ? fmaf(an, v - h, h) : fmaf(a, h, v);
}

template <class E, int V, bool BLEND> __global__ void __launch_bounds__(kBlock) k_scan_forward(ScanArgs a) {
    if (blockIdx.x >= a.piece_blocks) {
        if (blockIdx.y == 0) zero_unclaimed<E>(a, a.out0, nullptr);
        return;
    }
    Place p;
    if (!find_place<V>(a, p)) return;
    float h[V];
    if (p.is_head) load_state<V>(a.state, p.ray.id, a.C, p.c, h);
    else {
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = a.carry[(uint64_t)(p.begin / kPiece) * a.C + p.c + i];
    }
    for (uint32_t first = p.begin / kRows * kRows; first < p.end; first += kRows) {
        Block<E, V> g, v;
        g.load(a.gate, first, p.begin, p.end, a.C, p.c);
        v.load(a.value, first, p.begin, p.end, a.C, p.c);
        if (a.saved && first > p.ray.begin) store_f32<V>(a.saved, (uint64_t)(first / kRows) * a.C + p.c, h);
#pragma unroll
        for (uint32_t j = 0; j < kRows; ++j) {
            const uint32_t row = first + j;
            if (row < p.begin || row >= p.end) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float s, sn;
                sigmoid_pair(to_f32(g.r[j].v[i]), s, sn);
                h[i] = step<BLEND>(h[i], s, sn, to_f32(v.r[j].v[i]));
            }
            store_row<E, V>(a.out0, (uint64_t)row * a.C + p.c, h);
        }
    }
    if (p.end == p.ray.end && p.ray.id >= 0) store_f32<V>(a.last, (uint64_t)(uint32_t)p.ray.id * a.C + p.c, h);
}

template <class E, int V, bool BLEND> __global__ void __launch_bounds__(kBlock) k_scan_backward(ScanArgs a) {
    if (blockIdx.x >= a.piece_blocks) {
        if (blockIdx.y == 0) zero_unclaimed<E>(a, a.out0, a.out1);
        return;
    }
    Place p;
    if (!find_place<V>(a, p)) return;
    float e[V];
    if (p.end == p.ray.end) load_state<V>(a.dlast, p.ray.id, a.C, p.c, e);
    else {
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = a.carry[(uint64_t)(p.end / kPiece) * a.C + p.c + i];
    }
    const uint32_t first0 = p.begin / kRows * kRows;
    if (p.begin < p.end) {
        for (uint32_t first = (p.end - 1u) / kRows * kRows;; first -= kRows) {
            Block<E, V> g, v, d;
            g.load(a.gate, first, p.begin, p.end, a.C, p.c);
            v.load(a.value, first, p.begin, p.end, a.C, p.c);
            d.load(a.dh, first, p.begin, p.end, a.C, p.c);
            float h[V];
            if (first > p.ray.begin) {
#pragma unroll
                for (int i = 0; i < V; ++i) h[i] = a.saved[(uint64_t)(first / kRows) * a.C + p.c + i];
            } else load_state<V>(a.state, p.ray.id, a.C, p.c, h);
            float before[kRows][V];
#pragma unroll
            for (uint32_t j = 0; j < kRows; ++j) {
                const uint32_t row = first + j;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    before[j][i] = h[i];
                    float s, sn;
                    sigmoid_pair(to_f32(g.r[j].v[i]), s, sn);
                    const float next = step<BLEND>(h[i], s, sn, to_f32(v.r[j].v[i]));
                    h[i] = row >= p.begin ? next : h[i];
                }
            }
#pragma unroll
            for (uint32_t jj = 0; jj < kRows; ++jj) {
                const uint32_t j = kRows - 1u - jj, row = first + j;
                if (row < p.begin || row >= p.end) continue;
                float dg[V], dv[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float s, sn;
                    sigmoid_pair(to_f32(g.r[j].v[i]), s, sn);
                    const float G = to_f32(d.r[j].v[i]) + e[i], from = BLEND ? before[j][i] - to_f32(v.r[j].v[i]) : before[j][i];
                    dv[i] = BLEND ? G * sn : G;
                    dg[i] = G * from * (s * sn);
                    e[i] = s * G;
                }
                store_row<E, V>(a.out0, (uint64_t)row * a.C + p.c, dg);
                store_row<E, V>(a.out1, (uint64_t)row * a.C + p.c, dv);
            }
            if (first == first0) break;
        }
    }
    if (p.is_head && a.last && p.ray.id >= 0) store_f32<V>(a.last, (uint64_t)(uint32_t)p.ray.id * a.C + p.c, e);
}

// the affine map of the piece before border k (forward: what it does to h) or behind it (backward: what it does to E)
template <class E, int V, bool BLEND, bool BACK> __global__ void __launch_bounds__(kBlock) k_scan_sums(ScanArgs a) {
    const uint32_t per_block = kBlock / a.lanes, k = blockIdx.x * per_block + threadIdx.x / a.lanes;
    const uint32_t c = (blockIdx.y * a.lanes + (threadIdx.x & (a.lanes - 1u))) * V;
    RayRows ray;
    if (c >= a.C || border_owner(a, k, ray) < 0) return;
    const uint32_t begin = BACK ? k * kPiece : max(ray.begin, (k - 1u) * kPiece), end = BACK ? min(ray.end, (k + 1u) * kPiece) : k * kPiece;
    float A[V], B[V];
#pragma unroll
    for (int i = 0; i < V; ++i) { A[i] = 1.0f; B[i] = 0.0f; }
    const uint32_t first0 = begin / kRows * kRows, last0 = (end - 1u) / kRows * kRows;
    for (uint32_t first = BACK ? last0 : first0;; first = BACK ? first - kRows : first + kRows) {
        Block<E, V> g, v;
        g.load(a.gate, first, begin, end, a.C, c);
        v.load(BACK ? a.dh : a.value, first, begin, end, a.C, c);
#pragma unroll
        for (uint32_t jj = 0; jj < kRows; ++jj) {
            const uint32_t j = BACK ? kRows - 1u - jj : jj, row = first + j;
            const bool in = row >= begin && row < end;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float s, sn;
                sigmoid_pair(to_f32(g.r[j].v[i]), s, sn);
                const float x = to_f32(v.r[j].v[i]), b = BACK ? s * (B[i] + x) : step<BLEND>(B[i], s, sn, x);
                A[i] = in ? A[i] * s : A[i];
                B[i] = in ? b : B[i];
            }
        }
        if (first == (BACK ? first0 : last0)) break;
    }
    store_f32<V>(a.sum_a, (uint64_t)k * a.C + c, A);
    store_f32<V>(a.sum_b, (uint64_t)k * a.C + c, B);
}

// the maps of one cut ray's borders, joined in order.  The workgroup of the ray's first border works, the others leave.
template <bool BACK> __global__ void __launch_bounds__(kCarryThreads) k_scan_carry(ScanArgs a) {
    __shared__ float s_a[kCarryThreads], s_b[kCarryThreads];
    const uint32_t k0 = blockIdx.x;
    RayRows ray;
    if (border_owner(a, k0, ray) < 0 || ray.begin / kPiece + 1u != k0) return;          // (the same for the whole workgroup)
    const uint32_t borders = (ray.end - 1u) / kPiece - k0 + 1u;
    const uint32_t lane = threadIdx.x & (a.lanes - 1u), run = threadIdx.x / a.lanes, runs = kCarryThreads / a.lanes;
    const uint32_t c = blockIdx.y * a.lanes + lane;
    const bool on = c < a.C;
    const uint32_t each = (borders + runs - 1u) / runs, from = min(run * each, borders), to = min(from + each, borders);
    // position i of the order is border k0 + i forward, the last border - i backward
    auto at = [&](uint32_t i) { return (uint64_t)(BACK ? k0 + borders - 1u - i : k0 + i) * a.C + c; };
    float A = 1.0f, B = 0.0f;
    if (on) {
#pragma unroll 8
        for (uint32_t i = from; i < to; ++i) {
            const float x = a.sum_a[at(i)], y = a.sum_b[at(i)];
            B = fmaf(x, B, y);
            A *= x;
        }
    }
    s_a[threadIdx.x] = A;
    s_b[threadIdx.x] = B;
    __syncthreads();
    if (!on) return;
    const float* start = BACK ? a.dlast : a.state;
    float S = start && ray.id >= 0 ? start[(uint64_t)(uint32_t)ray.id * a.C + c] : 0.0f;
    for (uint32_t r = 0; r < run; ++r) S = fmaf(s_a[r * a.lanes + lane], S, s_b[r * a.lanes + lane]);
#pragma unroll 8
    for (uint32_t i = from; i < to; ++i) {
        S = fmaf(a.sum_a[at(i)], S, a.sum_b[at(i)]);
        a.carry[at(i)] = S;
    }
}

// the places of the workspace: sums and carries, then marks and owners when they are not kept in `saved`
uint64_t scan_tables(const ScanPlan& p, uint64_t T) { return round_up64(T, 4) + round_up64(p.borders, 4); }      // 4-byte words
uint64_t scan_sums_words(const ScanPlan& p, uint32_t C) { return 3ull * round_up64((uint64_t)p.borders * C, 4); }

template <class E, int V, bool BACK>
int launch_scan(ScanArgs a, int blend, void* workspace, float* saved, hipStream_t s) {
    const ScanPlan p = scan_plan<V>(a.T, a.N, a.C);
    float* w = static_cast<float*>(workspace);
    const uint64_t each = round_up64((uint64_t)p.borders * a.C, 4);
    a.sum_a = w;
    a.sum_b = w + each;
    a.carry = w + 2 * each;
    float* tables = saved ? saved + round_up64(p.states * a.C, 4) : w + 3 * each;
    a.mark = reinterpret_cast<int32_t*>(tables);
    a.owner = a.mark + round_up64(a.T, 4);
    a.saved = saved;
    a.cut = p.cut;
    a.borders = p.borders;
    a.lanes = p.lanes;
    const uint32_t per_block = kBlock / p.lanes;
    const uint64_t slots = (uint64_t)a.N + p.borders;
    a.piece_blocks = (uint32_t)((slots + per_block - 1) / per_block);
    const uint32_t zero_blocks = ceil_div(a.T, kBlock);          // (64 rows a wave)
    if (!BACK && a.N > 0) {
        hipLaunchKernelGGL(k_scan_map, dim3(ceil_div(a.N, kBlock / 64u)), dim3(kBlock), 0, s, a);
        if (int rc = check_launch("k_scan_map")) return rc;
    }
    if (p.cut) {
        const dim3 grid(ceil_div(p.borders, per_block), p.groups);
        if (blend) hipLaunchKernelGGL((k_scan_sums<E, V, true, BACK>), grid, dim3(kBlock), 0, s, a);
        else hipLaunchKernelGGL((k_scan_sums<E, V, false, BACK>), grid, dim3(kBlock), 0, s, a);
        if (int rc = check_launch("k_scan_sums")) return rc;
        ScanArgs b = a;
        const ScanPlan one = scan_plan<1>(a.T, a.N, a.C);
        b.lanes = one.lanes;
        hipLaunchKernelGGL((k_scan_carry<BACK>), dim3(p.borders, one.groups), dim3(kCarryThreads), 0, s, b);
        if (int rc = check_launch("k_scan_carry")) return rc;
    }
    const dim3 grid(a.piece_blocks + zero_blocks, p.groups);
    if constexpr (BACK) {
        if (blend) hipLaunchKernelGGL((k_scan_backward<E, V, true>), grid, dim3(kBlock), 0, s, a);
        else hipLaunchKernelGGL((k_scan_backward<E, V, false>), grid, dim3(kBlock), 0, s, a);
    } else {
        if (blend) hipLaunchKernelGGL((k_scan_forward<E, V, true>), grid, dim3(kBlock), 0, s, a);
        else hipLaunchKernelGGL((k_scan_forward<E, V, false>), grid, dim3(kBlock), 0, s, a);
    }
    return check_launch(BACK ? "k_scan_backward" : "k_scan_forward");
}

int scan_checks(const char* what, uint64_t T, uint32_t N, uint32_t C, int dtype, const void* workspace, uint64_t workspace_bytes) {
    ENVIDR_REQUIRE(dtype_ok(dtype), "%s: unknown dtype %d", what, dtype);
    ENVIDR_REQUIRE(C >= 1, "%s: no channels", what);
    ENVIDR_REQUIRE(T <= 0x7FFFFFFFull && N <= 0x7FFFFFFFu && C <= (1u << 20), "%s: T=%llu, N=%u or C=%u is too large", what, (unsigned long long)T, N, C);
    ENVIDR_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= envidr_ray_recurrence_workspace_bytes(T, N, C) && (workspace || T == 0),
                   "%s: workspace of %llu bytes, %llu needed", what, (unsigned long long)workspace_bytes, (unsigned long long)envidr_ray_recurrence_workspace_bytes(T, N, C));
    return ENVIDR_OK;
}

}  // namespace
}  // namespace envidr

using namespace envidr;

extern "C" {

uint64_t envidr_ray_recurrence_saved_floats(uint64_t T, uint32_t N, uint32_t C) {
    const ScanPlan p = scan_plan<1>(T, N, C);
    return round_up64(p.states * C, 4) + scan_tables(p, T);
}

uint64_t envidr_ray_recurrence_workspace_bytes(uint64_t T, uint32_t N, uint32_t C) {
    const ScanPlan p = scan_plan<1>(T, N, C);
    return 4ull * (scan_sums_words(p, C) + scan_tables(p, T));
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
    ENVIDR_FOR_DTYPE(dtype, E, { return (launch_scan<E, 1, false>(a, blend, workspace, saved, as_stream(stream))); });
}

int envidr_ray_recurrence_backward(const void* dh, const float* dlast, const void* gate, const void* value, const int32_t* rays,
                                   const float* state, const float* saved, uint64_t T, uint32_t N, uint32_t C, int dtype, int blend,
                                   void* dgate, void* dvalue, float* dstate, void* workspace, uint64_t workspace_bytes,
                                   envidr_stream_t stream) {
    if (int rc = scan_checks("ray_recurrence_backward", T, N, C, dtype, workspace, workspace_bytes)) return rc;
    if (N == 0 && T == 0) return ENVIDR_OK;
    ENVIDR_REQUIRE((dh && gate && value && saved && dgate && dvalue) || T == 0, "ray_recurrence_backward: null pointer");
    ENVIDR_REQUIRE(rays || N == 0, "ray_recurrence_backward: null pointer");
    ScanArgs a{};
    a.dh = dh; a.dlast = dlast; a.gate = gate; a.value = value; a.rays = rays; a.state = state; a.out0 = dgate; a.out1 = dvalue; a.last = dstate;
    a.T = (uint32_t)T; a.N = N; a.C = C;
    ENVIDR_FOR_DTYPE(dtype, E, { return (launch_scan<E, 1, true>(a, blend, workspace, const_cast<float*>(saved), as_stream(stream))); });
}

}  // extern "C"
