// recurrence.hip — gated linear recurrence over time-major sequences (B, T, C), channels contiguous (gfx950).
//
//   f = sigmoid(gate);  h_t = f_t h_{t-1} + u_t,   u_t = (1 - f_t) x_t (convex) or x_t (unit);  h_0 given or zero, channel by channel
//   g_t = dh_t + f_{t+1} g_{t+1} (the last live step also takes the gradient of the last state)
//   dx_t = (1 - f_t) g_t (convex) or g_t;  dgate_t = g_t (h_{t-1} - x_t or h_{t-1}) f_t (1 - f_t);  dh_0 = f_1 g_1
// `reverse` runs time from the last live row to the first.  Rows at or behind an item's length are not read and leave as zeros.
//
// Bound: HBM.  A step is a map h -> A h + U, and maps compose: a run of steps is one (A, U), so time is cut three ways.
//   * A thread takes V channels and L consecutive steps ("slot"), held in registers; it composes its own map.
//   * The slots of a workgroup make a tile: maps are scanned over a wave's slots by shuffles and over the waves through LDS; every thread then replays its steps
//     from its own entry state.  h itself never leaves fp32 before the store.
//   * A workgroup walks over the tiles of its item and channels with the state in registers, the next tile's loads in flight under the present one: one read,
//     one write.  Where items x channels leave too few workgroups for that (few long sequences), the tiles are also spread over workgroups: a first kernel leaves
//     each chunk's (A, U), the second starts each chunk from the maps before it; gates and inputs are read twice.
// 2 x 32768 x 1024 fp32 (8 chunks): maps 134 us (4.0 TB/s), forward 154 (5.2), gradient maps 126, backward 273 (4.9); one read of everything would take 430 us in all.
// Cutting the launches along time so that the second read meets the Infinity Cache does not shorten it (two halves: 80 + 71 us each, four quarters 43 + 35).
// 32 x 860 x 384 bf16 (no chunks): 21 + 36 us.
// The backward pass needs h_{t-1} in fp32 at every step: the forward leaves the state at every STATE_STEPS-th step, the backward rebuilds a tile from there
// (x and gate it reads anyway) and runs the gradient's recurrence, the same composition from the end.
#include "xva_common.h"
#include "../../include/xva_hip.h"
#include "seq_vec.h"

namespace {
using xva_seq::load_v;
using xva_seq::store_v;

constexpr int STATE_STEPS = 64;

struct Args {
    const void* x; const void* gate; void* h;              // (B, T, C)
    const float* h0; float* last;                          // (B, C)
    const void* dh; const float* dlast; void* dx; void* dgate; float* dh0;
    const int32_t* lens;
    float* states;                                         // (B, ceil(T / STATE_STEPS), C): the state before step i * STATE_STEPS; null: not wanted
    float* maps;                                           // split form: (B, chunks, 2, C): (A, U) of each chunk, U the forward's or the gradient's
    int64_t xb, xt, gb, gt, hb, ht, db, dt, dxb, dxt, dgb, dgt;
    int B, T, C, reverse, unit;
    int lc, lc_log, cblocks, tile, tiles, chunks, tiles_per_chunk, nstates;
    int near;                                              // the rows of a tile lie within 2^31 bytes
};

// f and 1 - f, each without cancellation, from one exponential that cannot overflow (a NaN stays one)
__device__ __forceinline__ void gates(float g, float& f, float& keep) {
    const float e = __expf(-fabsf(g)), big = __builtin_amdgcn_rcpf(1.f + e), small = e * big;
    f = g < 0.f ? small : big;
    keep = g < 0.f ? big : small;
}

typedef float f32x2 __attribute__((ext_vector_type(2)));
// V packed elements of type DT
template <int DT, int V> struct Raw {
    typedef typename std::conditional<DT == 0, typename std::conditional<V == 2, f32x2, float>::type, typename std::conditional<V == 2, uint32_t, uint16_t>::type>::type T;
    T v;
    __device__ __forceinline__ void get(float (&f)[V]) const {
        if constexpr (DT == 0) {
            if constexpr (V == 2) { f[0] = v[0]; f[1] = v[1]; } else f[0] = v;
        } else if constexpr (V == 2) xva_glds::unpack2<DT == 2>(v, f[0], f[1]);
        else f[0] = xva_glds::ld16<DT == 2>(&v, 0);
    }
};

// Where a thread is.  Step s = 0 .. len - 1 of time order is row s, or len - 1 - s in reverse.
struct Place {
    int b, c, slot, wave, waves, sub, subs, len;     // item, first channel, slot; wave, slots of a wave and which of them; live rows
    bool on;                                         // c < C
    int chunk, t0, t1;                               // tiles of this workgroup
    template <int V> static __device__ __forceinline__ Place make(const Args& a) {
        Place p;
        const int lane = threadIdx.x & 63;
        p.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); p.waves = blockDim.x >> 6;
        p.subs = 64 >> a.lc_log; p.sub = lane >> a.lc_log; p.slot = p.wave * p.subs + p.sub;
        // workgroups go to the eight XCDs by turns: neighbours in memory get the same one, so that a line they share is fetched once
        const int per = gridDim.x >> 3, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
        p.b = id / a.cblocks;
        const int c = ((id - p.b * a.cblocks) * a.lc + (lane & (a.lc - 1))) * V;
        p.on = c < a.C && p.b < a.B;
        p.c = p.on ? c : 0;
        p.b = min(p.b, a.B - 1);
        p.len = a.lens ? min(max(a.lens[p.b], 0), a.T) : a.T;
        p.chunk = blockIdx.y; p.t0 = p.chunk * a.tiles_per_chunk; p.t1 = min(p.t0 + a.tiles_per_chunk, a.tiles);
        return p;
    }
    __device__ __forceinline__ int64_t row(const Args& a, int s) const { return a.reverse ? len - 1 - s : s; }
};

// One tensor as a thread reads or writes it.  In a tile that is all live the address is a uniform row (scalar unit) plus this lane's fixed offset.
template <int DT, int V> struct Tensor {
    typedef typename Raw<DT, V>::T E;
    static constexpr int ES = DT == 0 ? 4 : 2;
    char* base;                                      // of the item
    int64_t st;                                      // bytes from row to row
    uint32_t off;
    int c;
    __device__ __forceinline__ Tensor(const Args& a, const Place& p, const void* t, int64_t sb, int64_t st_, int L) {
        base = (char*)t + p.b * sb * ES; st = st_ * ES; c = p.c * ES;
        off = (uint32_t)(a.reverse ? a.tile - L - p.slot * L : p.slot * L) * (uint32_t)st + (uint32_t)c;
    }
    // row of step k of a slot, less the lane's part: the tile's first step is `first`
    __device__ __forceinline__ char* uniform(const Args& a, const Place& p, int first, int k, int L) const {
        return base + (a.reverse ? (int64_t)(p.len - 1 - first - a.tile + L - k) : (int64_t)(first + k)) * st;
    }
    template <int L> __device__ __forceinline__ void fetch(const Args& a, const Place& p, int first, Raw<DT, V> (&r)[L]) const {
        if (a.near && first + a.tile <= p.len) {
#pragma unroll
            for (int k = 0; k < L; ++k) r[k].v = *reinterpret_cast<const E*>(uniform(a, p, first, k, L) + off);
        } else {                                     // steps behind the length stand still on the last live one (len >= 1)
            const int s0 = first + p.slot * L;
            const char* at = base + p.row(a, min(s0, p.len - 1)) * st + c;
#pragma unroll
            for (int k = 0; k < L; ++k) {
                r[k].v = *reinterpret_cast<const E*>(at);
                if (s0 + k + 1 < p.len) at += a.reverse ? -st : st;
            }
        }
    }
    template <bool FULL> __device__ __forceinline__ void store(const Args& a, const Place& p, int first, int k, int L, const float (&v)[V]) const {
        if constexpr (FULL) store_v<DT, V>(uniform(a, p, first, k, L) + off, 0, v);
        else {
            const int s = first + p.slot * L + k;
            if (s < p.len) store_v<DT, V>(base + p.row(a, s) * st + c, 0, v);
        }
    }
    __device__ __forceinline__ void zero(int row) const {
        const float z[V] = {};
        store_v<DT, V>(base + (int64_t)row * st + c, 0, z);
    }
};
// f and the input's weight of L steps; a step that is not there keeps the state: f = 1, weight 0
template <int DT, int V, int L, bool FULL>
__device__ __forceinline__ void weigh(const Place& p, int s0, const Raw<DT, V> (&r)[L], float (&f)[L][V], float (&keep)[L][V]) {
#pragma unroll
    for (int k = 0; k < L; ++k) {
        float g[V];
        r[k].get(g);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            gates(g[e], f[k][e], keep[k][e]);
            if (!FULL) {
                f[k][e] = s0 + k < p.len ? f[k][e] : 1.f;
                keep[k][e] = s0 + k < p.len ? keep[k][e] : 0.f;
            }
        }
    }
}
// values of L steps, nothing behind the length
template <int DT, int V, int L, bool FULL>
__device__ __forceinline__ void values(const Place& p, int s0, const Raw<DT, V> (&r)[L], float (&x)[L][V]) {
#pragma unroll
    for (int k = 0; k < L; ++k) {
        r[k].get(x[k]);
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (!FULL) x[k][e] = s0 + k < p.len ? x[k][e] : 0.f;
    }
}

// Maps of a wave's slots, scanned in time order (DIR > 0) or against it: (A, U) becomes the inclusive map from the wave's entry, (pA, pU) the one of the slots before
template <int V, int DIR>
__device__ __forceinline__ void scan_wave(const Args& a, const Place& p, float (&A)[V], float (&U)[V], float (&pA)[V], float (&pU)[V]) {
    const int lane = threadIdx.x & 63;
    const int pos = DIR > 0 ? p.sub : p.subs - 1 - p.sub;
    for (int o = 1; o < p.subs; o <<= 1) {
        const int from = DIR > 0 ? lane - o * a.lc : lane + o * a.lc;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float eA = __shfl(A[e], from & 63, 64), eU = __shfl(U[e], from & 63, 64);
            if (pos >= o) { U[e] = A[e] * eU + U[e]; A[e] *= eA; }
        }
    }
    const int from = DIR > 0 ? lane - a.lc : lane + a.lc;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const float eA = __shfl(A[e], from & 63, 64), eU = __shfl(U[e], from & 63, 64);
        pA[e] = pos > 0 ? eA : 1.f;
        pU[e] = pos > 0 ? eU : 0.f;
    }
}
__device__ __forceinline__ bool last_sub(const Place& p, int dir) { return dir > 0 ? p.sub == p.subs - 1 : p.sub == 0; }

// State of this wave's entry: the maps of the waves before it (DIR > 0) or behind it, from LDS [wave][lane of the channel][A, U], onto the tile's entry state h; with
// TO_END the rest follows, and h becomes the state behind the last
template <int V, int DIR, bool TO_END>
__device__ __forceinline__ void chain(const Args& a, const Place& p, const float* lds, float (&h)[V], float (&mine)[V]) {
    const float* at = lds + ((DIR > 0 ? 0 : p.waves - 1) * a.lc + (threadIdx.x & (a.lc - 1))) * 2 * V;
    const int step = (DIR > 0 ? a.lc : -a.lc) * 2 * V, before = DIR > 0 ? p.wave : p.waves - 1 - p.wave;
    auto apply = [&](int n, float (&s)[V]) __attribute__((always_inline)) {
        for (int i = 0; i < n; ++i) {
            float m[2 * V];
            if constexpr (V == 2) { const float4 t = *reinterpret_cast<const float4*>(at); m[0] = t.x; m[1] = t.y; m[2] = t.z; m[3] = t.w; }
            else { const float2 t = *reinterpret_cast<const float2*>(at); m[0] = t.x; m[1] = t.y; }
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] = m[e] * s[e] + m[V + e];
            at += step;
        }
    };
#pragma unroll
    for (int e = 0; e < V; ++e) mine[e] = h[e];
    apply(before, mine);
    if (TO_END) {
#pragma unroll
        for (int e = 0; e < V; ++e) h[e] = mine[e];
        apply(p.waves - before, h);
    }
}

// ================================================================================ forward ====
template <int DT, int V, int L>
__global__ __launch_bounds__(512, DT == 0 ? 2 : 4) void fwd_kernel(Args a) {
    extern __shared__ __attribute__((aligned(16))) float lds[];                 // [waves][lc][2 V]
    const Place p = Place::make<V>(a);
    float h[V];                                                                 // state at the tile's entry, the same in every slot
#pragma unroll
    for (int e = 0; e < V; ++e) h[e] = a.h0 ? a.h0[(int64_t)p.b * a.C + p.c + e] : 0.f;
    for (int k = 0; k < p.chunk; ++k) {
        const float* m = a.maps + ((int64_t)p.b * a.chunks + k) * 2 * a.C + p.c;
#pragma unroll
        for (int e = 0; e < V; ++e) h[e] = m[e] * h[e] + m[a.C + e];
    }
    const Tensor<DT, V> gate(a, p, a.gate, a.gb, a.gt, L), x(a, p, a.x, a.xb, a.xt, L), out(a, p, a.h, a.hb, a.ht, L);
    Raw<DT, V> rx[L], rg[L];
    if (p.t0 * a.tile < p.len) { gate.fetch(a, p, p.t0 * a.tile, rg); x.fetch(a, p, p.t0 * a.tile, rx); }
    auto one = [&](int tile, auto full) __attribute__((always_inline)) {
        constexpr bool FULL = decltype(full)::value;
        const int first = tile * a.tile, s0 = first + p.slot * L;
        float f[L][V], u[L][V], A[V], U[V], pA[V], pU[V], mine[V];
        {
            float keep[L][V];
            weigh<DT, V, L, FULL>(p, s0, rg, f, keep);
            values<DT, V, L, FULL>(p, s0, rx, u);
            if (!a.unit) {
#pragma unroll
                for (int k = 0; k < L; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e) u[k][e] *= keep[k][e];
            }
        }
        if (tile + 1 < p.t1 && first + a.tile < p.len) { gate.fetch(a, p, first + a.tile, rg); x.fetch(a, p, first + a.tile, rx); }
#pragma unroll
        for (int e = 0; e < V; ++e) { A[e] = 1.f; U[e] = 0.f; }
#pragma unroll
        for (int k = 0; k < L; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) { A[e] *= f[k][e]; U[e] = f[k][e] * U[e] + u[k][e]; }
        scan_wave<V, 1>(a, p, A, U, pA, pU);
        __syncthreads();                                                        // the maps of the tile before have been read
        if (last_sub(p, 1)) {
            float* m = lds + (p.wave * a.lc + (threadIdx.x & (a.lc - 1))) * 2 * V;
#pragma unroll
            for (int e = 0; e < V; ++e) { m[e] = A[e]; m[V + e] = U[e]; }
        }
        __syncthreads();
        chain<V, 1, true>(a, p, lds, h, mine);
#pragma unroll
        for (int e = 0; e < V; ++e) mine[e] = pA[e] * mine[e] + pU[e];
        if (p.on) {
            if (a.states && s0 % STATE_STEPS == 0 && s0 < a.T) store_v<0, V>(a.states, ((int64_t)p.b * a.nstates + s0 / STATE_STEPS) * a.C + p.c, mine);
#pragma unroll
            for (int k = 0; k < L; ++k) {
#pragma unroll
                for (int e = 0; e < V; ++e) mine[e] = f[k][e] * mine[e] + u[k][e];
                out.template store<FULL>(a, p, first, k, L, mine);
            }
        }
    };
    for (int tile = p.t0; tile < p.t1; ++tile) {
        const int first = tile * a.tile, s0 = first + p.slot * L;
        if (a.near && first + a.tile <= p.len) one(tile, std::true_type{});
        else {
            if (first < p.len) one(tile, std::false_type{});
            else if (a.states && p.on && s0 % STATE_STEPS == 0 && s0 < a.T) store_v<0, V>(a.states, ((int64_t)p.b * a.nstates + s0 / STATE_STEPS) * a.C + p.c, h);
            if (p.on)                                                           // rows behind the length follow the live ones in either direction
                for (int s = max(s0, p.len); s < min(s0 + L, a.T); ++s) out.zero(s);
        }
    }
    if (p.on && p.slot == 0 && p.t1 == a.tiles) store_v<0, V>(a.last, (int64_t)p.b * a.C + p.c, h);
}

// split form: the map of one chunk.  BWD: the gradient's map, from the chunk's end to its start
template <int DT, int V, int L, bool BWD>
__global__ __launch_bounds__(512) void map_kernel(Args a) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const Place p = Place::make<V>(a);
    constexpr int DIR = BWD ? -1 : 1;
    float tA[V], tU[V];                                                         // of the tiles so far
#pragma unroll
    for (int e = 0; e < V; ++e) { tA[e] = 1.f; tU[e] = 0.f; }
    const Tensor<DT, V> gate(a, p, a.gate, a.gb, a.gt, L), other(a, p, BWD ? a.dh : a.x, BWD ? a.db : a.xb, BWD ? a.dt : a.xt, L);
    const int live = min(p.t1, (p.len + a.tile - 1) / a.tile), n = live - p.t0;       // tiles with something in them
    Raw<DT, V> ru[L], rg[L];
    if (n > 0) { const int first = (BWD ? live - 1 : p.t0) * a.tile; gate.fetch(a, p, first, rg); other.fetch(a, p, first, ru); }
    auto one = [&](int first, bool more, auto full) __attribute__((always_inline)) {
        constexpr bool FULL = decltype(full)::value;
        const int s0 = first + p.slot * L;
        float f[L][V], u[L][V], A[V], U[V], pA[V], pU[V];
        {
            float keep[L][V];
            weigh<DT, V, L, FULL>(p, s0, rg, f, keep);
            values<DT, V, L, FULL>(p, s0, ru, u);
            if (!BWD && !a.unit) {
#pragma unroll
                for (int k = 0; k < L; ++k)
#pragma unroll
                    for (int e = 0; e < V; ++e) u[k][e] *= keep[k][e];
            }
        }
        if (more) { const int next = BWD ? first - a.tile : first + a.tile; gate.fetch(a, p, next, rg); other.fetch(a, p, next, ru); }
#pragma unroll
        for (int e = 0; e < V; ++e) { A[e] = 1.f; U[e] = 0.f; }
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int k = BWD ? L - 1 - i : i;
#pragma unroll
            for (int e = 0; e < V; ++e) { A[e] *= f[k][e]; U[e] = BWD ? f[k][e] * (U[e] + u[k][e]) : f[k][e] * U[e] + u[k][e]; }
        }
        scan_wave<V, DIR>(a, p, A, U, pA, pU);
        __syncthreads();
        if (last_sub(p, DIR)) {
            float* m = lds + (p.wave * a.lc + (threadIdx.x & (a.lc - 1))) * 2 * V;
#pragma unroll
            for (int e = 0; e < V; ++e) { m[e] = A[e]; m[V + e] = U[e]; }
        }
        __syncthreads();
        if (p.slot == 0)
            for (int i = 0; i < p.waves; ++i) {
                const float* m = lds + ((BWD ? p.waves - 1 - i : i) * a.lc + (threadIdx.x & (a.lc - 1))) * 2 * V;
#pragma unroll
                for (int e = 0; e < V; ++e) { tU[e] = m[e] * tU[e] + m[V + e]; tA[e] *= m[e]; }
            }
    };
    for (int i = 0; i < n; ++i) {
        const int first = (BWD ? live - 1 - i : p.t0 + i) * a.tile;
        if (a.near && first + a.tile <= p.len) one(first, i + 1 < n, std::true_type{});
        else one(first, i + 1 < n, std::false_type{});
    }
    if (p.on && p.slot == 0) {
        float* m = a.maps + ((int64_t)p.b * a.chunks + p.chunk) * 2 * a.C + p.c;
#pragma unroll
        for (int e = 0; e < V; ++e) { m[e] = tA[e]; m[a.C + e] = tU[e]; }
    }
}

// ================================================================================ backward ====
template <int DT, int V, int L>
__global__ __launch_bounds__(512) void bwd_kernel(Args a) {
    extern __shared__ __attribute__((aligned(16))) float lds[];                 // [waves][lc][A, U], then [waves][lc][A, W]: the states' and the gradient's maps
    const Place p = Place::make<V>(a);
    float q[V];                                                                 // f_{t+1} g_{t+1} at the tile's end
#pragma unroll
    for (int e = 0; e < V; ++e) q[e] = a.dlast ? a.dlast[(int64_t)p.b * a.C + p.c + e] : 0.f;
    for (int k = a.chunks - 1; k > p.chunk; --k) {
        const float* m = a.maps + ((int64_t)p.b * a.chunks + k) * 2 * a.C + p.c;
#pragma unroll
        for (int e = 0; e < V; ++e) q[e] = m[e] * q[e] + m[a.C + e];
    }
    const Tensor<DT, V> gate(a, p, a.gate, a.gb, a.gt, L), x(a, p, a.x, a.xb, a.xt, L), grad(a, p, a.dh, a.db, a.dt, L);
    const Tensor<DT, V> dx(a, p, a.dx, a.dxb, a.dxt, L), dgate(a, p, a.dgate, a.dgb, a.dgt, L);
    const int live = min(p.t1, (p.len + a.tile - 1) / a.tile);                  // tiles t0 .. live - 1 have something in them
    Raw<DT, V> rx[L], rg[L], rd[L];
    auto fetch = [&](int tile) __attribute__((always_inline)) { gate.fetch(a, p, tile * a.tile, rg); x.fetch(a, p, tile * a.tile, rx); grad.fetch(a, p, tile * a.tile, rd); };
    if (live > p.t0) fetch(live - 1);
    auto one = [&](int tile, auto full) __attribute__((always_inline)) {
        constexpr bool FULL = decltype(full)::value;
        const int first = tile * a.tile, s0 = first + p.slot * L;
        float f[L][V], keep[L][V], v[L][V], dh[L][V], A[V], U[V], W[V], B[V], pA[V], pU[V], sA[V], sW[V], h[V], hm[V], mine[V];
        load_v<0, V>(a.states, ((int64_t)p.b * a.nstates + tile * (a.tile / STATE_STEPS)) * a.C + p.c, h);
        weigh<DT, V, L, FULL>(p, s0, rg, f, keep);
        values<DT, V, L, FULL>(p, s0, rx, v);
        values<DT, V, L, FULL>(p, s0, rd, dh);
        if (tile > p.t0) fetch(tile - 1);
#pragma unroll
        for (int e = 0; e < V; ++e) { A[e] = 1.f; U[e] = 0.f; W[e] = 0.f; }
#pragma unroll
        for (int k = 0; k < L; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) { A[e] *= f[k][e]; U[e] = f[k][e] * U[e] + (a.unit ? v[k][e] : keep[k][e] * v[k][e]); }
#pragma unroll
        for (int k = L - 1; k >= 0; --k)
#pragma unroll
            for (int e = 0; e < V; ++e) W[e] = f[k][e] * (W[e] + dh[k][e]);
#pragma unroll
        for (int e = 0; e < V; ++e) B[e] = A[e];
        scan_wave<V, 1>(a, p, A, U, pA, pU);
        scan_wave<V, -1>(a, p, B, W, sA, sW);
        __syncthreads();
        float* m = lds + (p.wave * a.lc + (threadIdx.x & (a.lc - 1))) * 2 * V;
        float* mW = m + p.waves * a.lc * 2 * V;
        if (last_sub(p, 1)) {
#pragma unroll
            for (int e = 0; e < V; ++e) { m[e] = A[e]; m[V + e] = U[e]; }
        }
        if (last_sub(p, -1)) {
#pragma unroll
            for (int e = 0; e < V; ++e) { mW[e] = B[e]; mW[V + e] = W[e]; }
        }
        __syncthreads();
        chain<V, 1, false>(a, p, lds, h, hm);
        chain<V, -1, true>(a, p, lds + p.waves * a.lc * 2 * V, q, mine);
        if (p.on) {
#pragma unroll
            for (int e = 0; e < V; ++e) { hm[e] = pA[e] * hm[e] + pU[e]; mine[e] = sA[e] * mine[e] + sW[e]; }
            // v becomes what the gate pulls at: h_{t-1} - x_t (convex) or h_{t-1}
#pragma unroll
            for (int k = 0; k < L; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float now = v[k][e], before = hm[e];
                    hm[e] = f[k][e] * before + (a.unit ? now : keep[k][e] * now);
                    v[k][e] = a.unit ? before : before - now;
                }
#pragma unroll
            for (int k = L - 1; k >= 0; --k) {
                float ox[V], og[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float g = mine[e] + dh[k][e];
                    ox[e] = a.unit ? g : keep[k][e] * g;
                    mine[e] = f[k][e] * g;
                    og[e] = mine[e] * keep[k][e] * v[k][e];
                }
                dx.template store<FULL>(a, p, first, k, L, ox);
                dgate.template store<FULL>(a, p, first, k, L, og);
            }
        }
    };
    for (int tile = live - 1; tile >= p.t0; --tile) {
        if (a.near && (tile + 1) * a.tile <= p.len) one(tile, std::true_type{});
        else one(tile, std::false_type{});
    }
    if (p.on) {
        for (int s = max(p.len, p.t0 * a.tile) + p.slot; s < min(a.T, p.t1 * a.tile); s += p.waves * p.subs) { dx.zero(s); dgate.zero(s); }
        if (p.slot == 0 && p.t0 == 0 && a.dh0) store_v<0, V>(a.dh0, (int64_t)p.b * a.C + p.c, q);
    }
}

// -------------------------------------------------------------------------------- plan ----
constexpr int L_FWD = 8, L_BWD = 8;      // steps of a slot: what the registers of 512 threads hold

int state_count(int T) { return T > 0 ? (T + STATE_STEPS - 1) / STATE_STEPS : 1; }

struct Plan { int v, lc, lc_log, threads, tile, tiles, chunks, tiles_per_chunk, cblocks; };

Plan make_plan(int dtype, int B, int T, int C, int v, bool bwd) {
    Plan p;
    p.v = v;
    const int lanes = (C + v - 1) / v;
    // lanes of channels in a wave (the rest of it are slots): 64, less where there are no more channels, or down to 16 (half a line of 16-bit values, whose
    // other half is the neighbour's) where that gives workgroups to CUs without one.  32 x 860 x 384 bf16 forward: 192 workgroups of 32 lanes 24 us, 384 of 16 21 us.
    int lc = 64;
    while (lc > 1 && lc / 2 >= lanes) lc /= 2;
    while (lc > 16 && (int64_t)B * ((lanes + lc - 1) / lc) < 256) lc /= 2;
    // Still few: rows of 32 bytes, where that fills the CUs and time need not be cut, so that inputs are read once.  Kernels' time, us, cut | narrow: 32 x 3000 x 64 fp32
    // forward 36 | 20, backward 43 | 31; 2 x 3000 x 1024 37 | 22, 44 | 32; 1 x 8192 x 4096 bf16 74 | 57, 118 | 113; longer than that the cut wins or draws (4 x 16384 x 512
    // fp32 131 | 141, 190 | 207).
    const int narrow = 32 / (v * (dtype == 0 ? 4 : 2));
    if (T <= 8192 && (int64_t)B * ((lanes + lc - 1) / lc) < 160 && narrow < lc && (int64_t)B * ((lanes + narrow - 1) / narrow) >= 256) lc = narrow;
    p.lc = lc;
    p.lc_log = __builtin_ctz(lc);
    p.cblocks = (lanes + lc - 1) / lc;
    // waves: no more than the sequence has use for; whole tiles of STATE_STEPS (or one tile that holds everything)
    const int wave_steps = 64 / lc * (bwd ? L_BWD : L_FWD);
    int waves = (int)(((int64_t)T + wave_steps - 1) / wave_steps);
    if (waves > 8) waves = 8;
    if (waves < 1) waves = 1;
    p.tile = waves * wave_steps;
    p.threads = waves * 64;
    p.tiles = T > 0 ? (T + p.tile - 1) / p.tile : 1;
    // Split time where items x channels leave CUs without work.  2 x 32768 x 1024 fp32, forward + backward: one workgroup to 8 lanes and all of time (128 of them)
    // 325 + 541 us, 64 of 16 lanes cut into 8 chunks 290 + 399 us though inputs are read twice; at 192 workgroups (above) the one read wins.
    const int64_t wgs = (int64_t)B * p.cblocks;
    int64_t chunks = wgs >= 160 ? 1 : (512 + wgs - 1) / wgs;
    if (chunks > p.tiles) chunks = p.tiles;
    if (chunks > 256) chunks = 256;
    p.tiles_per_chunk = (int)((p.tiles + chunks - 1) / chunks);
    p.chunks = (p.tiles + p.tiles_per_chunk - 1) / p.tiles_per_chunk;
    return p;
}
int64_t map_floats(const Plan& q, int B, int C) { return q.chunks > 1 ? (int64_t)B * q.chunks * 2 * C : 0; }
int64_t workspace(int B, int T, int C) {
    int64_t most = 0;               // over the types and widths that the call may turn out to have
    for (int dtype = 0; dtype < 2; ++dtype)
        for (int v = 1; v <= 2; ++v)
            for (int bwd = 0; bwd < 2; ++bwd) {
                const int64_t n = v == 2 && C % 2 ? 0 : map_floats(make_plan(dtype, B, T, C, v, bwd != 0), B, C);
                if (n > most) most = n;
            }
    return most * 4;
}

// two channels to a lane (one where C, a stride or an address is odd)
int vec_of(const xva_recurrence_args* p, bool bwd) {
    const int es = xva_seq::elem_size(p->dtype);
    int64_t all = p->C | p->x_stride[0] | p->x_stride[1] | p->gate_stride[0] | p->gate_stride[1];
    uintptr_t ptrs = (uintptr_t)p->x | (uintptr_t)p->gate;
    if (!bwd) { all |= p->h_stride[0] | p->h_stride[1]; ptrs |= (uintptr_t)p->h; }
    else {
        all |= p->dh_stride[0] | p->dh_stride[1] | p->dx_stride[0] | p->dx_stride[1] | p->dgate_stride[0] | p->dgate_stride[1];
        ptrs |= (uintptr_t)p->dh | (uintptr_t)p->dx | (uintptr_t)p->dgate;
    }
    const uintptr_t wide = (uintptr_t)p->states | (uintptr_t)p->last | (uintptr_t)p->dh0;
    return all % 2 == 0 && ptrs % (2 * es) == 0 && wide % 8 == 0 ? 2 : 1;
}

template <int DT, int V> int launch(const Args& a, const Plan& q, bool bwd, hipStream_t st) {
    const dim3 grid((unsigned)((a.B * q.cblocks + 7) / 8 * 8), q.chunks);
    const size_t lds = (size_t)(q.threads / 64) * q.lc * V * 4;
    if (!bwd) {
        if (q.chunks > 1) {
            map_kernel<DT, V, L_FWD, false><<<grid, q.threads, 2 * lds, st>>>(a);
            XVA_LAUNCH_CHECK();
        }
        fwd_kernel<DT, V, L_FWD><<<grid, q.threads, 2 * lds, st>>>(a);
    } else {
        if (q.chunks > 1) {
            map_kernel<DT, V, L_BWD, true><<<grid, q.threads, 2 * lds, st>>>(a);
            XVA_LAUNCH_CHECK();
        }
        bwd_kernel<DT, V, L_BWD><<<grid, q.threads, 4 * lds, st>>>(a);
    }
    XVA_LAUNCH_CHECK();
    return XVA_OK;
}

int run(const xva_recurrence_args* p, bool bwd, void* ws, int64_t ws_bytes, void* stream, const char* who) {
    XVA_CHECK_ARG(p, "%s: null argument", who);
    XVA_CHECK_ARG(p->dtype >= 0 && p->dtype <= 2, "%s: dtype %d", who, p->dtype);
    XVA_CHECK_ARG(p->B >= 0 && p->T >= 0 && p->T < (1 << 30) && p->C >= 1 && (int64_t)p->B * p->C < (1ll << 31), "%s: B %d T %d C %d", who, p->B, p->T, p->C);
    XVA_CHECK_ARG((int64_t)p->C * xva_seq::elem_size(p->dtype) < (1ll << 31), "%s: C %d, rows are under 2^31 bytes", who, p->C);        // (32-bit offsets in a row)
    if (p->B == 0) return XVA_OK;
    XVA_CHECK_ARG(p->T == 0 || (p->x && p->gate), "%s: null argument", who);
    XVA_CHECK_ARG(bwd ? p->states && (p->T == 0 || (p->dh && p->dx && p->dgate)) : p->last && (p->T == 0 || p->h), "%s: null argument", who);
    const Plan q = make_plan(p->dtype, p->B, p->T, p->C, vec_of(p, bwd), bwd);
    XVA_CHECK_ARG(xva_seq::launchable(((int64_t)p->B * q.cblocks + 7) / 8 * 8, q.threads), "%s: B %d T %d C %d: too many items", who, p->B, p->T, p->C);
    const int64_t need = map_floats(q, p->B, p->C) * 4;
    if (ws_bytes < need || (need && !ws)) { xva_set_error("%s: workspace of %lld bytes, %lld needed", who, (long long)ws_bytes, (long long)need); return XVA_ERR_WS; }
    Args a = {};
    a.x = p->x; a.gate = p->gate; a.h = p->h; a.h0 = p->h0; a.last = p->last; a.dh = p->dh; a.dlast = p->dlast; a.dx = p->dx; a.dgate = p->dgate; a.dh0 = p->dh0;
    a.lens = p->lens; a.states = p->states; a.maps = (float*)ws;
    a.xb = p->x_stride[0]; a.xt = p->x_stride[1]; a.gb = p->gate_stride[0]; a.gt = p->gate_stride[1]; a.hb = p->h_stride[0]; a.ht = p->h_stride[1];
    a.db = p->dh_stride[0]; a.dt = p->dh_stride[1]; a.dxb = p->dx_stride[0]; a.dxt = p->dx_stride[1]; a.dgb = p->dgate_stride[0]; a.dgt = p->dgate_stride[1];
    a.B = p->B; a.T = p->T; a.C = p->C; a.reverse = p->reverse; a.unit = p->unit_gain;
    a.lc = q.lc; a.lc_log = q.lc_log; a.cblocks = q.cblocks; a.tile = q.tile; a.tiles = q.tiles; a.chunks = q.chunks; a.tiles_per_chunk = q.tiles_per_chunk;
    a.nstates = state_count(p->T);
    a.near = 1;
    for (int64_t e : {a.xt, a.gt, a.ht, a.dt, a.dxt, a.dgt}) if (e < 0 || e * q.tile >= (1ll << 29)) a.near = 0;
    hipStream_t st = (hipStream_t)stream;
    if (p->dtype == 0) return q.v == 2 ? launch<0, 2>(a, q, bwd, st) : launch<0, 1>(a, q, bwd, st);
    if (p->dtype == 1) return q.v == 2 ? launch<1, 2>(a, q, bwd, st) : launch<1, 1>(a, q, bwd, st);
    return q.v == 2 ? launch<2, 2>(a, q, bwd, st) : launch<2, 1>(a, q, bwd, st);
}
}   // namespace

extern "C" int64_t xva_recurrence_workspace_bytes(int B, int T, int C) { return B < 0 || T < 0 || C < 1 ? -1 : (B == 0 ? 0 : workspace(B, T, C)); }
extern "C" int64_t xva_recurrence_state_floats(int B, int T, int C) {
    if (B < 0 || T < 0 || C < 1) return -1;
    return (int64_t)B * C * state_count(T);
}
extern "C" int xva_recurrence_fwd(const xva_recurrence_args* p, void* ws, int64_t ws_bytes, void* stream) { return run(p, false, ws, ws_bytes, stream, "xva_recurrence_fwd"); }
extern "C" int xva_recurrence_bwd(const xva_recurrence_args* p, void* ws, int64_t ws_bytes, void* stream) { return run(p, true, ws, ws_bytes, stream, "xva_recurrence_bwd"); }
