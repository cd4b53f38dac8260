// recurrence.hip — gated linear recurrence over time-major sequences (B, T, C), channels contiguous (gfx950).
//
//   f = sigmoid(gate);  h_t = f_t h_{t-1} + u_t,   u_t = (1 - f_t) x_t (convex) or x_t (unit);  h_0 given or zero, channel by channel
//   g_t = dh_t + f_{t+1} g_{t+1} (the last live step also takes the gradient of the last state)
//   dx_t = (1 - f_t) g_t (convex) or g_t;  dgate_t = g_t (h_{t-1} - x_t or h_{t-1}) f_t (1 - f_t);  dh_0 = f_1 g_1
// `reverse` runs time from the last live row to the first.  Rows at or behind an item's length are not read and leave as zeros.
//
// Bound: HBM.  A step is a map h -> A h + U, and maps compose: a run of steps is one (A, U), so time is cut three ways.
//   * A thread takes V channels and L consecutive steps ("slot"), held in registers; it composes its own map.
//   * The slots of a workgroup (a tile of S x L steps) exchange their maps through LDS; every thread applies those before its own to the tile's entry state
//     and replays its steps from there.  h itself never leaves fp32 before the store.
//   * Where items x channels alone fill the card, a workgroup walks over the tiles of its item, the state in registers (one read, one write).  Where they
//     do not (few long sequences), the tiles are spread over workgroups: a first kernel leaves each chunk's (A, U), the second starts each chunk from the
//     maps before it; the gates and inputs are read twice.
// The backward pass needs h_{t-1} in fp32 at every step: the forward leaves the state at each tile's entry, the backward rebuilds the tile from there
// (x and gate it reads anyway) and runs the gradient's recurrence, the same composition from the end.
#include "xva_common.h"
#include "../../include/xva_hip.h"
#include "seq_vec.h"

namespace {
using xva_seq::load_v;
using xva_seq::store_v;

struct Args {
    const void* x; const void* gate; void* h;              // (B, T, C)
    const float* h0; float* last;                          // (B, C)
    const void* dh; const float* dlast; void* dx; void* dgate; float* dh0;
    const int32_t* lens;
    float* states;                                         // (B, tiles, C): the state at each tile's entry; null: not wanted
    float* maps;                                           // split form: (B, chunks, 2, C): (A, U) of each chunk, U the forward's or the gradient's
    int64_t xb, xt, gb, gt, hb, ht, db, dt, dxb, dxt, dgb, dgt;
    int B, T, C, reverse, unit;
    int lc, slots, tiles, chunks, tiles_per_chunk;
};

// f and 1 - f, each without cancellation, from one exponential that cannot overflow (a NaN stays one)
__device__ __forceinline__ void gates(float g, float& f, float& keep) {
    const float e = __expf(-fabsf(g)), big = __builtin_amdgcn_rcpf(1.f + e), small = e * big;
    f = g < 0.f ? small : big;
    keep = g < 0.f ? big : small;
}

// step s = 0 .. len - 1 of time order is row s, or len - 1 - s in reverse
__device__ __forceinline__ int64_t row_of(const Args& a, int len, int s) { return a.reverse ? len - 1 - s : s; }

template <int DT, int V, int L>
__device__ __forceinline__ void read_steps(const Args& a, const void* base, int64_t sb, int64_t st, int b, int c, int len, int s0, bool on, float (&f)[L][V]) {
#pragma unroll
    for (int k = 0; k < L; ++k) {
        if (on && s0 + k < len) load_v<DT, V>(base, b * sb + row_of(a, len, s0 + k) * st + c, f[k]);
        else {
#pragma unroll
            for (int e = 0; e < V; ++e) f[k][e] = 0.f;
        }
    }
}

// What every kernel here starts with: its item, channels and slot.  lds: [slots][lc][2 (or 3)][V]
#define XVA_REC_PLACE                                                                                             \
    const int lane = threadIdx.x % a.lc, slot = threadIdx.x / a.lc;                                               \
    const int cblocks = (a.C / V + a.lc - 1) / a.lc;                                                              \
    const int cb = blockIdx.x % cblocks, b = blockIdx.x / cblocks;                                                \
    const int c = (cb * a.lc + lane) * V;                                                                         \
    const bool on = slot < a.slots && c < a.C;                                                                    \
    const int len = a.lens ? min(max(a.lens[b], 0), a.T) : a.T;                                                   \
    const int tile_steps = a.slots * L;

// (A, U) of the steps in f, u
template <int V, int L> __device__ __forceinline__ void compose(const float (&f)[L][V], const float (&u)[L][V], float (&A)[V], float (&U)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) { A[e] = 1.f; U[e] = 0.f; }
#pragma unroll
    for (int k = 0; k < L; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) { A[e] *= f[k][e]; U[e] = f[k][e] * U[e] + u[k][e]; }
}

// gates and inputs of L steps; a step that is not there keeps the state: f = 1, u = 0
template <int DT, int V, int L>
__device__ __forceinline__ void steps_of(const Args& a, int b, int c, int len, int s0, bool on, float (&f)[L][V], float (&u)[L][V]) {
    read_steps<DT, V, L>(a, a.gate, a.gb, a.gt, b, c, len, s0, on, f);
    read_steps<DT, V, L>(a, a.x, a.xb, a.xt, b, c, len, s0, on, u);
#pragma unroll
    for (int k = 0; k < L; ++k) {
        const bool there = on && s0 + k < len;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float ff, keep;
            gates(f[k][e], ff, keep);
            f[k][e] = there ? ff : 1.f;
            if (!a.unit) u[k][e] = there ? keep * u[k][e] : 0.f;
        }
    }
}

// ================================================================================ forward ====
template <int DT, int V, int L>
__global__ __launch_bounds__(1024) void fwd_kernel(Args a) {
    extern __shared__ float lds[];
    XVA_REC_PLACE
    const int chunk = blockIdx.y, t0 = chunk * a.tiles_per_chunk, t1 = min(t0 + a.tiles_per_chunk, a.tiles);
    float h[V];                                  // state at the tile's entry, the same in every slot
#pragma unroll
    for (int e = 0; e < V; ++e) h[e] = on && a.h0 ? a.h0[(int64_t)b * a.C + c + e] : 0.f;
    if (on)
        for (int k = 0; k < chunk; ++k) {
            const float* m = a.maps + ((int64_t)b * a.chunks + k) * 2 * a.C + c;
#pragma unroll
            for (int e = 0; e < V; ++e) h[e] = m[e] * h[e] + m[a.C + e];
        }
    for (int tile = t0; tile < t1; ++tile) {
        const int s0 = tile * tile_steps + slot * L;
        float f[L][V], u[L][V], A[V], U[V];
        steps_of<DT, V, L>(a, b, c, len, s0, on, f, u);
        compose<V, L>(f, u, A, U);
        if (a.states && on && slot == 0) store_v<0, V>(a.states, ((int64_t)b * a.tiles + tile) * a.C + c, h);
        __syncthreads();                         // the maps of the tile before have been read
        if (slot < a.slots) {
            float* m = lds + (slot * a.lc + lane) * 2 * V;
#pragma unroll
            for (int e = 0; e < V; ++e) { m[e] = A[e]; m[V + e] = U[e]; }
        }
        __syncthreads();
        float mine[V];
#pragma unroll
        for (int e = 0; e < V; ++e) mine[e] = h[e];
        for (int k = 0; k < a.slots; ++k) {
            const float* m = lds + (k * a.lc + lane) * 2 * V;
            if (k == slot) {
#pragma unroll
                for (int e = 0; e < V; ++e) mine[e] = h[e];
            }
#pragma unroll
            for (int e = 0; e < V; ++e) h[e] = m[e] * h[e] + m[V + e];
        }
        if (on) {
#pragma unroll
            for (int k = 0; k < L; ++k) {
                const int s = s0 + k;
                if (s >= a.T) break;
#pragma unroll
                for (int e = 0; e < V; ++e) mine[e] = f[k][e] * mine[e] + u[k][e];
                float out[V];
#pragma unroll
                for (int e = 0; e < V; ++e) out[e] = s < len ? mine[e] : 0.f;
                // (rows behind the length follow the live ones in either direction)
                store_v<DT, V>(a.h, b * a.hb + (s < len ? row_of(a, len, s) : s) * a.ht + c, out);
            }
        }
    }
    if (on && slot == 0 && t1 == a.tiles) store_v<0, V>(a.last, (int64_t)b * a.C + c, h);
}

// split form: the map of one chunk.  BWD: the gradient's map, from the chunk's end to its start
template <int DT, int V, int L, bool BWD>
__global__ __launch_bounds__(1024) void map_kernel(Args a) {
    extern __shared__ float lds[];
    XVA_REC_PLACE
    const int chunk = blockIdx.y, t0 = chunk * a.tiles_per_chunk, t1 = min(t0 + a.tiles_per_chunk, a.tiles);
    float tA[V], tU[V];
#pragma unroll
    for (int e = 0; e < V; ++e) { tA[e] = 1.f; tU[e] = 0.f; }
    for (int i = 0; i < t1 - t0; ++i) {
        const int tile = BWD ? t1 - 1 - i : t0 + i;
        const int s0 = tile * tile_steps + slot * L;
        float f[L][V], u[L][V], A[V], U[V];
        if constexpr (BWD) {
            read_steps<DT, V, L>(a, a.gate, a.gb, a.gt, b, c, len, s0, on, f);
            read_steps<DT, V, L>(a, a.dh, a.db, a.dt, b, c, len, s0, on, u);
#pragma unroll
            for (int e = 0; e < V; ++e) { A[e] = 1.f; U[e] = 0.f; }
#pragma unroll
            for (int k = L - 1; k >= 0; --k) {
                const bool there = on && s0 + k < len;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    float ff, keep;
                    gates(f[k][e], ff, keep);
                    ff = there ? ff : 1.f;
                    A[e] *= ff; U[e] = ff * (U[e] + u[k][e]);
                }
            }
        } else {
            steps_of<DT, V, L>(a, b, c, len, s0, on, f, u);
            compose<V, L>(f, u, A, U);
        }
        __syncthreads();
        if (slot < a.slots) {
            float* m = lds + (slot * a.lc + lane) * 2 * V;
#pragma unroll
            for (int e = 0; e < V; ++e) { m[e] = A[e]; m[V + e] = U[e]; }
        }
        __syncthreads();
        if (on && slot == 0)
            for (int k = 0; k < a.slots; ++k) {
                const float* m = lds + ((BWD ? a.slots - 1 - k : k) * a.lc + lane) * 2 * V;
#pragma unroll
                for (int e = 0; e < V; ++e) { tU[e] = m[e] * tU[e] + m[V + e]; tA[e] *= m[e]; }
            }
    }
    if (on && slot == 0) {
        float* m = a.maps + ((int64_t)b * a.chunks + chunk) * 2 * a.C + c;
#pragma unroll
        for (int e = 0; e < V; ++e) { m[e] = tA[e]; m[a.C + e] = tU[e]; }
    }
}

// ================================================================================ backward ====
template <int DT, int V, int L>
__global__ __launch_bounds__(1024) void bwd_kernel(Args a) {
    extern __shared__ float lds[];
    XVA_REC_PLACE
    const int chunk = blockIdx.y, t0 = chunk * a.tiles_per_chunk, t1 = min(t0 + a.tiles_per_chunk, a.tiles);
    float q[V];                                  // f_{t+1} g_{t+1} at the tile's end
#pragma unroll
    for (int e = 0; e < V; ++e) q[e] = on && a.dlast ? a.dlast[(int64_t)b * a.C + c + e] : 0.f;
    if (on)
        for (int k = a.chunks - 1; k > chunk; --k) {
            const float* m = a.maps + ((int64_t)b * a.chunks + k) * 2 * a.C + c;
#pragma unroll
            for (int e = 0; e < V; ++e) q[e] = m[e] * q[e] + m[a.C + e];
        }
    for (int tile = t1 - 1; tile >= t0; --tile) {
        const int s0 = tile * tile_steps + slot * L;
        float f[L][V], x[L][V], dh[L][V], A[V], U[V], W[V];
        read_steps<DT, V, L>(a, a.gate, a.gb, a.gt, b, c, len, s0, on, f);
        read_steps<DT, V, L>(a, a.x, a.xb, a.xt, b, c, len, s0, on, x);
        read_steps<DT, V, L>(a, a.dh, a.db, a.dt, b, c, len, s0, on, dh);
        float h[V];
#pragma unroll
        for (int e = 0; e < V; ++e) { A[e] = 1.f; U[e] = 0.f; W[e] = 0.f; h[e] = 0.f; }
        if (on) load_v<0, V>(a.states, ((int64_t)b * a.tiles + tile) * a.C + c, h);
        float keep[L][V];
#pragma unroll
        for (int k = 0; k < L; ++k) {
            const bool there = on && s0 + k < len;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float ff, kk;
                gates(f[k][e], ff, kk);
                f[k][e] = there ? ff : 1.f; keep[k][e] = there ? kk : 0.f;
                A[e] *= f[k][e];
                U[e] = f[k][e] * U[e] + (a.unit ? x[k][e] : keep[k][e] * x[k][e]);
            }
        }
#pragma unroll
        for (int k = L - 1; k >= 0; --k)
#pragma unroll
            for (int e = 0; e < V; ++e) W[e] = f[k][e] * (W[e] + dh[k][e]);
        __syncthreads();
        if (slot < a.slots) {
            float* m = lds + (slot * a.lc + lane) * 3 * V;
#pragma unroll
            for (int e = 0; e < V; ++e) { m[e] = A[e]; m[V + e] = U[e]; m[2 * V + e] = W[e]; }
        }
        __syncthreads();
        for (int k = 0; k < slot; ++k) {
            const float* m = lds + (k * a.lc + lane) * 3 * V;
#pragma unroll
            for (int e = 0; e < V; ++e) h[e] = m[e] * h[e] + m[V + e];
        }
        float mine[V];
#pragma unroll
        for (int e = 0; e < V; ++e) mine[e] = q[e];
        for (int k = a.slots - 1; k >= 0; --k) {
            const float* m = lds + (k * a.lc + lane) * 3 * V;
            if (k == slot) {
#pragma unroll
                for (int e = 0; e < V; ++e) mine[e] = q[e];
            }
#pragma unroll
            for (int e = 0; e < V; ++e) q[e] = m[e] * q[e] + m[2 * V + e];
        }
        if (on) {
            // x becomes what the gate pulls at: h_{t-1} - x_t (convex) or h_{t-1}
#pragma unroll
            for (int k = 0; k < L; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float now = x[k][e], before = h[e];
                    h[e] = f[k][e] * before + (a.unit ? now : keep[k][e] * now);
                    x[k][e] = a.unit ? before : before - now;
                }
#pragma unroll
            for (int k = L - 1; k >= 0; --k) {
                const int s = s0 + k;
                if (s >= a.T) continue;
                float dx[V], dg[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float g = mine[e] + dh[k][e];
                    dx[e] = s < len ? (a.unit ? g : keep[k][e] * g) : 0.f;
                    dg[e] = s < len ? g * x[k][e] * f[k][e] * keep[k][e] : 0.f;
                    mine[e] = f[k][e] * g;
                }
                const int64_t r = s < len ? row_of(a, len, s) : s;
                store_v<DT, V>(a.dx, b * a.dxb + r * a.dxt + c, dx);
                store_v<DT, V>(a.dgate, b * a.dgb + r * a.dgt + c, dg);
            }
        }
    }
    if (on && slot == 0 && t0 == 0 && a.dh0) store_v<0, V>(a.dh0, (int64_t)b * a.C + c, q);
}

// -------------------------------------------------------------------------------- plan ----
constexpr int L_STEPS = 8, MAX_SLOTS = 16;

// steps of a tile: what the states stand for, so a matter of the length alone (not of the widths that an address allows)
int tile_steps(int T) {
    const int slots = (T + L_STEPS - 1) / L_STEPS;
    return L_STEPS * (slots < 1 ? 1 : (slots < MAX_SLOTS ? slots : MAX_SLOTS));
}

struct Plan { int v, lc, slots, threads, tiles, chunks, tiles_per_chunk, cblocks; };

Plan make_plan(int B, int T, int C, int v) {
    Plan p;
    p.v = v;
    const int lanes = C / v;
    p.lc = lanes < 64 ? lanes : 64;
    p.cblocks = (lanes + p.lc - 1) / p.lc;
    p.slots = tile_steps(T) / L_STEPS;
    p.threads = (p.slots * p.lc + 63) / 64 * 64;
    p.tiles = T > 0 ? (T + tile_steps(T) - 1) / tile_steps(T) : 1;
    // split time where items x channels leave CUs without work: two workgroups to a CU wanted
    const int64_t wgs = (int64_t)B * p.cblocks;
    int64_t chunks = (512 + wgs - 1) / wgs;
    if (chunks > p.tiles) chunks = p.tiles;
    if (chunks > 256) chunks = 256;
    p.tiles_per_chunk = (int)((p.tiles + chunks - 1) / chunks);
    p.chunks = (p.tiles + p.tiles_per_chunk - 1) / p.tiles_per_chunk;
    return p;
}
int64_t workspace(int B, int T, int C) {
    int64_t most = 0;
    for (int v = 1; v <= 2; ++v) {
        if (C % v) continue;
        const Plan q = make_plan(B, T, C, v);
        const int64_t n = q.chunks > 1 ? (int64_t)B * q.chunks * 2 * C * 4 : 0;
        if (n > most) most = n;
    }
    return most;
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
    const dim3 grid((unsigned)(a.B * q.cblocks), q.chunks);
    const size_t lds = (size_t)q.slots * q.lc * V * 4;
    if (!bwd) {
        if (q.chunks > 1) {
            map_kernel<DT, V, L_STEPS, false><<<grid, q.threads, 2 * lds, st>>>(a);
            XVA_LAUNCH_CHECK();
        }
        fwd_kernel<DT, V, L_STEPS><<<grid, q.threads, 2 * lds, st>>>(a);
    } else {
        if (q.chunks > 1) {
            map_kernel<DT, V, L_STEPS, true><<<grid, q.threads, 2 * lds, st>>>(a);
            XVA_LAUNCH_CHECK();
        }
        bwd_kernel<DT, V, L_STEPS><<<grid, q.threads, 3 * lds, st>>>(a);
    }
    XVA_LAUNCH_CHECK();
    return XVA_OK;
}

int run(const xva_recurrence_args* p, bool bwd, void* ws, int64_t ws_bytes, void* stream, const char* who) {
    XVA_CHECK_ARG(p, "%s: null argument", who);
    XVA_CHECK_ARG(p->dtype >= 0 && p->dtype <= 2, "%s: dtype %d", who, p->dtype);
    XVA_CHECK_ARG(p->B >= 0 && p->T >= 0 && p->T < (1 << 30) && p->C >= 1 && (int64_t)p->B * p->C < (1ll << 31), "%s: B %d T %d C %d", who, p->B, p->T, p->C);
    if (p->B == 0) return XVA_OK;
    XVA_CHECK_ARG(p->T == 0 || (p->x && p->gate), "%s: null argument", who);
    XVA_CHECK_ARG(bwd ? p->states && (p->T == 0 || (p->dh && p->dx && p->dgate)) : p->last && (p->T == 0 || p->h), "%s: null argument", who);
    const Plan q = make_plan(p->B, p->T, p->C, vec_of(p, bwd));
    const int64_t need = q.chunks > 1 ? (int64_t)p->B * q.chunks * 2 * p->C * 4 : 0;
    if (ws_bytes < need || (need && !ws)) { xva_set_error("%s: workspace of %lld bytes, %lld needed", who, (long long)ws_bytes, (long long)need); return XVA_ERR_WS; }
    Args a = {};
    a.x = p->x; a.gate = p->gate; a.h = p->h; a.h0 = p->h0; a.last = p->last; a.dh = p->dh; a.dlast = p->dlast; a.dx = p->dx; a.dgate = p->dgate; a.dh0 = p->dh0;
    a.lens = p->lens; a.states = p->states; a.maps = (float*)ws;
    a.xb = p->x_stride[0]; a.xt = p->x_stride[1]; a.gb = p->gate_stride[0]; a.gt = p->gate_stride[1]; a.hb = p->h_stride[0]; a.ht = p->h_stride[1];
    a.db = p->dh_stride[0]; a.dt = p->dh_stride[1]; a.dxb = p->dx_stride[0]; a.dxt = p->dx_stride[1]; a.dgb = p->dgate_stride[0]; a.dgt = p->dgate_stride[1];
    a.B = p->B; a.T = p->T; a.C = p->C; a.reverse = p->reverse; a.unit = p->unit_gain;
    a.lc = q.lc; a.slots = q.slots; a.tiles = q.tiles; a.chunks = q.chunks; a.tiles_per_chunk = q.tiles_per_chunk;
    hipStream_t st = (hipStream_t)stream;
    if (p->dtype == 0) return q.v == 2 ? launch<0, 2>(a, q, bwd, st) : launch<0, 1>(a, q, bwd, st);
    if (p->dtype == 1) return q.v == 2 ? launch<1, 2>(a, q, bwd, st) : launch<1, 1>(a, q, bwd, st);
    return q.v == 2 ? launch<2, 2>(a, q, bwd, st) : launch<2, 1>(a, q, bwd, st);
}
}   // namespace

extern "C" int64_t xva_recurrence_workspace_bytes(int B, int T, int C) { return B < 0 || T < 0 || C < 1 ? -1 : (B == 0 ? 0 : workspace(B, T, C)); }
extern "C" int64_t xva_recurrence_state_floats(int B, int T, int C) {
    if (B < 0 || T < 0 || C < 1) return -1;
    return (int64_t)B * C * (T > 0 ? (T + tile_steps(T) - 1) / tile_steps(T) : 1);
}
extern "C" int xva_recurrence_fwd(const xva_recurrence_args* p, void* ws, int64_t ws_bytes, void* stream) { return run(p, false, ws, ws_bytes, stream, "xva_recurrence_fwd"); }
extern "C" int xva_recurrence_bwd(const xva_recurrence_args* p, void* ws, int64_t ws_bytes, void* stream) { return run(p, true, ws, ws_bytes, stream, "xva_recurrence_bwd"); }
