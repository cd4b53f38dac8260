// group_norm.hip — group normalisation with an activation over time-major sequences (B, T, C), channels contiguous (gfx950).
//
//   item b, group g of n = C / G channels, N = lens[b] * n live values:
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, z = xh w + bias, y = act(z)
//   dz = dy act'(z);  dw = sum dz xh, dbias = sum dz (over items and rows);  dx = r (w dz - mean(w dz) - xh mean(w dz xh))
// Rows at or behind an item's length count for nothing: they are not read, and leave as zeros.
//
// Bound: HBM (a training pass moves 5 tensors; the tile form 8, at 5.2 TB/s: 64 x 8192 x 32 fp32, 4 groups, gelu: statistics 14 us, result 24, sums of dz 29 + 5,
// dx 34, dw / dbias 4).  In the other forms latency: 27520 rows of 8 heads of 64 bf16: 14 + 22 + 4 us; 32 x 860 x 384 bf16, 16 groups, silu: 15 + 25 + 4 us (256
// workgroups whose registers leave room for one to a CU: it reads, reduces and writes one after the other), below the host's time for the pass.
// Three forms, by the size of one (item, group) slab of T x n values:
//   * slab: it fits the registers of (part of) one wave — each head's norm behind an attention (T = 1), short items.  A slab lies over a power of two of lanes, so
//     every reduction is a few shuffles; x is read once.  dw / dbias stay in the lanes' registers over all the items that a workgroup passes, leave as one partial
//     row per workgroup and are added in a fixed order.
//   * whole: some groups of an item fit the registers of a workgroup: read once, kept packed, normalised from there; one kernel forward, one and the sum of
//     dw / dbias over items backward.
//   * tile: chunks of rows (all channels of a row, so loads are whole lines whatever n is): statistics of each chunk, then one pass that joins them and writes.  x is
//     read twice forward, x and dy twice backward.
// Statistics are two-pass from registers and joined by the exact update of mean and squared deviations (Chan, Golub, LeVeque), so a mean that is large against the
// deviation costs nothing.  Everything is held in fp32; sums over rows are made in a fixed order, so results repeat bit for bit.
#include "xva_common.h"
#include "../../include/xva_hip.h"
#include "seq_vec.h"

namespace {
using xva_seq::Packed;
using xva_seq::lanes_sum;
using xva_seq::load_v;
using xva_seq::store_v;

enum { NONE, RELU, LRELU, TANH, SILU, GELU };

struct Args {
    const void* x; const void* dy; void* out;              // out: y or dx
    const float* w; const float* bias;
    const int32_t* lens;
    float* mean; float* rstd;                              // (B, G)
    float* part;                                           // partial results of the first kernel
    float* item;                                           // (B, 2, C): sums of dz and dz xh of each item
    float* dw; float* db;
    int64_t xb, xt, db_, dt_, ob, ot;                      // strides of x, dy and out
    int B, T, C, G, n, act;
    float eps, slope;
    int rows_per_chunk, chunks;
};

__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }
// (1 - e) / (1 + e) of |z|, e = exp(-2 |z|), whose difference of near numbers loses nothing that matters from 0.45 on; below, where small weights put z, the Taylor series
// (its next term is under 2^-25 of z there).  Some units of 2^-24 of itself everywhere.  (The library's tanhf, inlined for every value of the register forms, makes
// all their activations slower: 32 x 860 x 384 bf16 with silu 14.8 -> 16.7 us.)
__device__ __forceinline__ float tanh_(float z) {
    const float x = fabsf(z), q = z * z, e = __expf(-2.f * x), d = 1.f + e, r0 = __builtin_amdgcn_rcpf(d), r = __builtin_fmaf(__builtin_fmaf(-d, r0, 1.f), r0, r0);
    float p = 21844.f / 6081075.f;
    p = __builtin_fmaf(p, q, -1382.f / 155925.f);
    p = __builtin_fmaf(p, q, 62.f / 2835.f);
    p = __builtin_fmaf(p, q, -17.f / 315.f);
    p = __builtin_fmaf(p, q, 2.f / 15.f);
    p = __builtin_fmaf(p, q, -1.f / 3.f);
    return x < 0.45f ? __builtin_fmaf(p * q, z, z) : copysignf((1.f - e) * r, z);
}
// tanh'(z) = 4 e / (1 + e)^2, e = exp(-2 |z|): no difference of near numbers, at any z
__device__ __forceinline__ float tanh_slope(float z) {
    const float e = __expf(-2.f * fabsf(z)), r = __builtin_amdgcn_rcpf(1.f + e);
    return 4.f * e * r * r;
}
// (one switch to V values: a branch of every value costs more than the activations)
template <int V, class F> __device__ __forceinline__ void each(float (&z)[V], F f) {
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] = f(z[e]);
}
template <int V> __device__ __forceinline__ void activate(float (&z)[V], int act, float slope) {
    switch (act) {
        case RELU: each<V>(z, [](float v) { return v > 0.f ? v : (v != v ? v : 0.f); }); break;
        case LRELU: each<V>(z, [=](float v) { return v > 0.f ? v : slope * v; }); break;
        case TANH: each<V>(z, [](float v) { return tanh_(v); }); break;
        case SILU: each<V>(z, [](float v) { return v * sigmoid(v); }); break;
        case GELU: each<V>(z, [](float v) { return 0.5f * v * (1.f + erff(v * 0.70710678118654752f)); }); break;
        default: break;
    }
}
// z -> act'(z)
template <int V> __device__ __forceinline__ void slopes(float (&z)[V], int act, float slope) {
    switch (act) {
        case RELU: each<V>(z, [](float v) { return v > 0.f ? 1.f : 0.f; }); break;
        case LRELU: each<V>(z, [=](float v) { return v > 0.f ? 1.f : slope; }); break;
        case TANH: each<V>(z, [](float v) { return tanh_slope(v); }); break;
        case SILU: each<V>(z, [](float v) { const float s = sigmoid(v); return s + s * v * (1.f - s); }); break;
        case GELU: each<V>(z, [](float v) { return 0.5f * (1.f + erff(v * 0.70710678118654752f)) + v * 0.39894228040143268f * __expf(-0.5f * v * v); }); break;
        default: each<V>(z, [](float) { return 1.f; });
    }
}
// V values of a weight vector, `none` where there is none.  Vectors of 32-bit values are loaded from any address of one (a slice of a flat parameter buffer), so the
// weights' address has no say in how x is read.
template <int V> __device__ __forceinline__ void load_w(const float* w, int c, float none, float (&f)[V]) {
    typedef float Any __attribute__((ext_vector_type(V < 4 ? V : 4), aligned(4)));
    if (w) {
#pragma unroll
        for (int e = 0; e < V; e += 4) {
            const Any v = *reinterpret_cast<const Any*>(w + c + e);
#pragma unroll
            for (int i = 0; i < (V < 4 ? V : 4); ++i) f[e + i] = v[i];
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = none;
    }
}
__device__ __forceinline__ int live_rows(const Args& a, int b) {
    return a.lens ? min(max(a.lens[b], 0), a.T) : a.T;
}
// ================================================================================ slab form ====
// LPG lanes hold one slab, NV vectors of V values each: vector j = k * LPG + lane of the slab is row j / (n / V), channels (j % (n / V)) * V ...
// A workgroup holds 256 / LPG slabs: GPB groups of 256 / (LPG * GPB) items, and walks over the items.
struct SlabPlan { int lpg, gpb, ipb, gy; };

template <int DT, int V, int NV, bool BWD>
__global__ __launch_bounds__(256) void slab_kernel(Args a, SlabPlan s) {
    extern __shared__ float sums[];                        // BWD: [256 lanes][NV][2][V]
    const int lane = threadIdx.x & (s.lpg - 1), slot = threadIdx.x / s.lpg;
    const int gl = slot % s.gpb, il = slot / s.gpb;
    const int g = blockIdx.y * s.gpb + gl;
    const bool mine = il < s.ipb && g < a.G;
    const int nv = a.n / V, vecs = a.T * nv;
    int row[NV], ch[NV];
    float w[NV][V], bias[NV][V], sw[NV][V], sb[NV][V];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int j = k * s.lpg + lane;
        row[k] = j < vecs ? j / nv : a.T;                  // a.T: no such row
        ch[k] = min(g, a.G - 1) * a.n + (j < vecs ? (j % nv) * V : 0);
        load_w<V>(a.w, ch[k], 1.f, w[k]);
        load_w<V>(a.bias, ch[k], 0.f, bias[k]);
#pragma unroll
        for (int e = 0; e < V; ++e) sw[k][e] = sb[k][e] = 0.f;
    }
    // this item's values, and the next one's on their way
    Packed<DT, V> nx[NV], ng[NV];
    int nlen = 0;
    auto fetch = [&](int64_t b) __attribute__((always_inline)) {
        nlen = mine && b < a.B ? live_rows(a, (int)b) : 0;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            nx[k].clear();
            if (BWD) ng[k].clear();
            if (row[k] < nlen) {
                nx[k].load(a.x, b * a.xb + (int64_t)row[k] * a.xt + ch[k]);
                if (BWD) ng[k].load(a.dy, b * a.db_ + (int64_t)row[k] * a.dt_ + ch[k]);
            }
        }
    };
    const int64_t step = (int64_t)gridDim.x * s.ipb;
    fetch((int64_t)blockIdx.x * s.ipb + il);
    for (int64_t b0 = (int64_t)blockIdx.x * s.ipb; b0 < a.B; b0 += step) {
        const int64_t b = b0 + il;
        const bool on = mine && b < a.B;
        const int len = nlen;
        float x[NV][V], dz[NV][V];
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            nx[k].get(x[k]);
            if (BWD) ng[k].get(dz[k]);
#pragma unroll
            for (int e = 0; e < V; ++e) sum += x[k][e];
        }
        if (b0 + step < a.B) fetch(b + step);
        const float inv_n = len > 0 ? 1.f / ((float)len * (float)a.n) : 0.f;
        float mean, rstd;
        if constexpr (!BWD) {
            mean = lanes_sum(sum, s.lpg) * inv_n;
            float sq = 0.f;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < V; ++e) { const float d = row[k] < len ? x[k][e] - mean : 0.f; sq += d * d; }
            rstd = rsqrtf(lanes_sum(sq, s.lpg) * inv_n + a.eps);
            if (on && lane == 0) { a.mean[b * a.G + g] = mean; a.rstd[b * a.G + g] = rstd; }
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (!on || row[k] >= a.T) continue;
                float z[V];
#pragma unroll
                for (int e = 0; e < V; ++e) z[e] = (x[k][e] - mean) * rstd * w[k][e] + bias[k][e];
                activate<V>(z, a.act, a.slope);
                if (row[k] >= len) {
#pragma unroll
                    for (int e = 0; e < V; ++e) z[e] = 0.f;
                }
                store_v<DT, V>(a.out, b * a.ob + (int64_t)row[k] * a.ot + ch[k], z);
            }
        } else {
            mean = on ? a.mean[b * a.G + g] : 0.f;
            rstd = on ? a.rstd[b * a.G + g] : 0.f;
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                float z[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    x[k][e] = row[k] < len ? (x[k][e] - mean) * rstd : 0.f;
                    z[e] = x[k][e] * w[k][e] + bias[k][e];
                }
                slopes<V>(z, a.act, a.slope);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float xh = x[k][e], d = dz[k][e] * z[e];
                    sw[k][e] += d * xh; sb[k][e] += d;
                    dz[k][e] = d * w[k][e];
                    s1 += dz[k][e]; s2 += dz[k][e] * xh;
                }
            }
            s1 = lanes_sum(s1, s.lpg) * inv_n;
            s2 = lanes_sum(s2, s.lpg) * inv_n;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (!on || row[k] >= a.T) continue;
                float d[V];
#pragma unroll
                for (int e = 0; e < V; ++e) d[e] = row[k] < len ? rstd * (dz[k][e] - s1 - x[k][e] * s2) : 0.f;
                store_v<DT, V>(a.out, b * a.ob + (int64_t)row[k] * a.ot + ch[k], d);
            }
        }
    }
    if constexpr (BWD) {
        // the lanes that hold one channel (its items and rows) are added in a fixed order: partial row (blockIdx.x) of (2, C)
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                sums[((threadIdx.x * NV + k) * 2) * V + e] = mine ? sb[k][e] : 0.f;
                sums[((threadIdx.x * NV + k) * 2 + 1) * V + e] = mine ? sw[k][e] : 0.f;
            }
        __syncthreads();
        for (int c = threadIdx.x; c < s.gpb * a.n; c += 256) {
            const int cg = c / a.n, cc = c - cg * a.n, v = cc / V, e = cc - v * V;
            if (blockIdx.y * s.gpb + cg >= a.G) continue;
            float t1 = 0.f, t2 = 0.f;
            for (int i = 0; i < s.ipb; ++i)
                for (int r = 0; r < a.T; ++r) {
                    const int j = r * nv + v, k = j / s.lpg, th = (i * s.gpb + cg) * s.lpg + j - k * s.lpg;
                    t1 += sums[((th * NV + k) * 2) * V + e];
                    t2 += sums[((th * NV + k) * 2 + 1) * V + e];
                }
            const int c_all = blockIdx.y * s.gpb * a.n + c;
            a.part[((int64_t)blockIdx.x * 2) * a.C + c_all] = t1;
            a.part[((int64_t)blockIdx.x * 2 + 1) * a.C + c_all] = t2;
        }
    }
}

// ================================================================================ whole form ====
// A workgroup holds all T rows of `gpw` groups of an item: lv vectors of a row side by side, threads / lv rows at once, NV vectors to a thread.  A vector lies in one
// group (n is a multiple of V).
struct WholePlan { int threads, gpw, lv, rows, blocks; };

// sums over the workgroup of one value a thread, group by group: red[threads], result in out[gpw]
__device__ __forceinline__ void whole_sums(float v, float* red, float* out, const WholePlan& q, int nv) {
    red[threadIdx.x] = v;
    __syncthreads();
    const int lane = threadIdx.x & 63, waves = q.threads >> 6, count = q.rows * nv;
    for (int g = threadIdx.x >> 6; g < q.gpw; g += waves) {
        float t = 0.f;
        for (int i = lane; i < count; i += 64) { const int r = i / nv; t += red[r * q.lv + g * nv + i - r * nv]; }
        t = lanes_sum(t, 64);
        if (lane == 0) out[g] = t;
    }
    __syncthreads();
}

template <int DT, int V, int NV, bool BWD>
__global__ __launch_bounds__(512) void whole_kernel(Args a, WholePlan q) {
    extern __shared__ float lds[];                 // threads | 2 gpw; backward: rows * channels instead of threads, and 2 x channels
    // workgroups go to the eight XCDs by turns: those that share an item's lines get the same one
    const int per = gridDim.x >> 3, id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    const int b = id / q.blocks, blk = id - b * q.blocks;
    if (b >= a.B) return;
    const int r0 = threadIdx.x / q.lv, v = threadIdx.x - r0 * q.lv;
    const int nv = a.n / V, g0 = blk * q.gpw, gn = min(q.gpw, a.G - g0), gl = v / nv, g = g0 + gl;
    const bool on = r0 < q.rows && gl < gn;
    const int len = live_rows(a, b), c = g0 * a.n + v * V;
    const float inv_n = len > 0 ? 1.f / ((float)len * (float)a.n) : 0.f;
    Packed<DT, V> x[NV], d[BWD ? NV : 1];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int r = r0 + k * q.rows;
        x[k].clear();
        if (BWD) d[k].clear();
        if (on && r < len) {
            x[k].load(a.x, b * a.xb + (int64_t)r * a.xt + c);
            if (BWD) d[k].load(a.dy, b * a.db_ + (int64_t)r * a.dt_ + c);
        }
    }
    float w[V], bias[V];
    load_w<V>(a.w, on ? c : 0, 1.f, w);
    load_w<V>(a.bias, on ? c : 0, 0.f, bias);
    if constexpr (!BWD) {
        float* sums = lds + q.threads;
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float f[V];
            x[k].get(f);
#pragma unroll
            for (int e = 0; e < V; ++e) s += f[e];
        }
        whole_sums(s, lds, sums, q, nv);
        const float mean = sums[min(gl, q.gpw - 1)] * inv_n;
        s = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float f[V];
            x[k].get(f);
            if (r0 + k * q.rows < len) {
#pragma unroll
                for (int e = 0; e < V; ++e) s += (f[e] - mean) * (f[e] - mean);
            }
        }
        whole_sums(on ? s : 0.f, lds, sums + q.gpw, q, nv);
        const float rstd = rsqrtf(sums[q.gpw + min(gl, q.gpw - 1)] * inv_n + a.eps);
        if (on && r0 == 0 && v == gl * nv) { a.mean[(int64_t)b * a.G + g] = mean; a.rstd[(int64_t)b * a.G + g] = rstd; }
        // four vectors to a switch over the activations: each one's code follows on itself
#pragma unroll
        for (int k0 = 0; k0 < NV; k0 += 4) {
            if (!on || r0 + k0 * q.rows >= a.T) continue;
            float z[4 * V];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float f[V];
                x[k0 + k].get(f);
#pragma unroll
                for (int e = 0; e < V; ++e) z[k * V + e] = (f[e] - mean) * rstd * w[e] + bias[e];
            }
            activate<4 * V>(z, a.act, a.slope);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int r = r0 + (k0 + k) * q.rows;
                if (r >= a.T) continue;
                float f[V];
#pragma unroll
                for (int e = 0; e < V; ++e) f[e] = r < len ? z[k * V + e] : 0.f;
                store_v<DT, V>(a.out, b * a.ob + (int64_t)r * a.ot + c, f);
            }
        }
    } else {
        const int cw = q.lv * V;                   // channels of the workgroup
        float* ch = lds + q.rows * cw;             // [2][channels]: sums of dz, dz xh
        float* sums = ch + 2 * cw;                 // [2][gpw]
        const float mean = on ? a.mean[(int64_t)b * a.G + g] : 0.f, rstd = on ? a.rstd[(int64_t)b * a.G + g] : 0.f;
        float s1[V], s2[V];
#pragma unroll
        for (int e = 0; e < V; ++e) s1[e] = s2[e] = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (r0 + k * q.rows >= len) continue;
            float f[V], h[V], z[V];
            x[k].get(f); d[k].get(h);
#pragma unroll
            for (int e = 0; e < V; ++e) { f[e] = (f[e] - mean) * rstd; z[e] = f[e] * w[e] + bias[e]; }
            slopes<V>(z, a.act, a.slope);
#pragma unroll
            for (int e = 0; e < V; ++e) { const float dz = h[e] * z[e]; s1[e] += dz; s2[e] += dz * f[e]; }
        }
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            if (r0 < q.rows) {
#pragma unroll
                for (int e = 0; e < V; ++e) lds[r0 * cw + v * V + e] = which ? s2[e] : s1[e];
            }
            __syncthreads();
            // a few threads to a channel, each a share of the rows; neighbours in a run of lanes add up
            int run = 1;
            while (run < 16 && run * 2 * cw <= q.threads) run *= 2;
            for (int c0 = 0; c0 < cw; c0 += q.threads / run) {
                const int cc = c0 + threadIdx.x / run;
                float t = 0.f;
                if (cc < cw)
                    for (int r = threadIdx.x & (run - 1); r < q.rows; r += run) t += lds[r * cw + cc];
                t = lanes_sum(t, run);
                if (cc < cw && (threadIdx.x & (run - 1)) == 0) {
                    ch[which * cw + cc] = t;
                    if (cc < gn * a.n) a.part[((int64_t)b * 2 + which) * a.C + g0 * a.n + cc] = t;
                }
            }
            __syncthreads();
        }
        const int lane = threadIdx.x & 63, waves = q.threads >> 6;
        for (int i = threadIdx.x >> 6; i < 2 * gn; i += waves) {
            const int which = i / gn, gg = i - which * gn;
            float t = 0.f;
            for (int cc = gg * a.n + lane; cc < (gg + 1) * a.n; cc += 64) t += (a.w ? a.w[g0 * a.n + cc] : 1.f) * ch[which * cw + cc];
            t = lanes_sum(t, 64);
            if (lane == 0) sums[which * q.gpw + gg] = t * inv_n;
        }
        __syncthreads();
        const float k1 = sums[min(gl, q.gpw - 1)], k2 = sums[q.gpw + min(gl, q.gpw - 1)];
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int r = r0 + k * q.rows;
            if (!on || r >= a.T) continue;
            float f[V], h[V], z[V];
            x[k].get(f); d[k].get(h);
#pragma unroll
            for (int e = 0; e < V; ++e) { f[e] = (f[e] - mean) * rstd; z[e] = f[e] * w[e] + bias[e]; }
            slopes<V>(z, a.act, a.slope);
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = r < len ? rstd * (w[e] * (h[e] * z[e]) - k1 - f[e] * k2) : 0.f;
            store_v<DT, V>(a.out, b * a.ob + (int64_t)r * a.ot + c, f);
        }
    }
}

// ================================================================================ tile form ====
// A thread owns one vector of V channels and every `step`-th row of its chunk; lc = C / V vectors side by side, step = blockDim.x / lc rows at once.
constexpr int NR = 8;      // rows of a thread in one register tile
constexpr int MAX_CHUNKS = 256;        // of an item

struct Tile {
    int lc, step, v, r; bool on;
    __device__ __forceinline__ Tile(int C, int V) {
        lc = C / V; step = blockDim.x / lc;
        r = threadIdx.x / lc; v = threadIdx.x - r * lc;
        on = r < step;
    }
};
// per-thread sums -> red[row slot][channel]
template <int V> __device__ __forceinline__ void put(float* red, const Tile& t, int C, const float (&s)[V]) {
    if (t.on) {
#pragma unroll
        for (int e = 0; e < V; ++e) red[t.r * C + t.v * V + e] = s[e];
    }
}
// Runs of lanes that share a sum: `chans` lanes over the n channels of a group (a power of two), times as many over the row slots as keep all groups within one turn
// of the workgroup (few channels mean many slots).
struct Run { int chans, lanes; };
__device__ __forceinline__ Run run_of(int n, int G, int slots) {
    Run r = {1, 1};
    while (r.chans < n && r.chans < 64) r.chans <<= 1;
    r.lanes = r.chans;
    while (r.lanes < 64 && 2 * r.lanes * G <= (int)blockDim.x && r.lanes < r.chans * slots) r.lanes <<= 1;
    return r;
}
// group sums of red into out[g]
__device__ __forceinline__ void group_sums(const float* red, float* out, const Tile& t, int C, int G, int n, Run run) {
    const int per = blockDim.x / run.lanes, lane = threadIdx.x & (run.lanes - 1), cl = lane & (run.chans - 1), s0 = lane / run.chans, ss = run.lanes / run.chans;
    for (int g0 = 0; g0 < G; g0 += per) {
        const int g = g0 + threadIdx.x / run.lanes;
        float v = 0.f;
        if (g < G)
            for (int sl = s0; sl < t.step; sl += ss)
                for (int c = cl; c < n; c += run.chans) v += red[sl * C + g * n + c];
        v = lanes_sum(v, run.lanes);
        if (g < G && lane == 0) out[g] = v;
    }
}

// statistics of one chunk: part[(b * chunks + chunk) * G + g] = (mean, sum of squared deviations)
template <int DT, int V, int NT>
__global__ __launch_bounds__(NT) void tile_stats_kernel(Args a) {
    extern __shared__ float lds[];
    const Tile t(a.C, V);
    float* red = lds;                          // step * C
    float* mean = red + t.step * a.C;          // G: running mean, then squared deviations
    float* m2 = mean + a.G;
    float* now = m2 + a.G;                     // G: this tile's sums
    const int b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks, len = live_rows(a, b);
    const Run run = run_of(a.n, a.G, t.step);
    const int first = chunk * a.rows_per_chunk, end = min(first + a.rows_per_chunk, len);
    for (int g = threadIdx.x; g < a.G; g += blockDim.x) mean[g] = m2[g] = 0.f;
    float before = 0.f;                        // rows joined so far
    int mine[V];                               // groups of this thread's channels
#pragma unroll
    for (int e = 0; e < V; ++e) mine[e] = t.on ? (t.v * V + e) / a.n : 0;
    const int64_t base = (int64_t)b * a.xb + t.v * V;
    for (int r0 = first; r0 < end; r0 += t.step * NR) {
        float f[NR][V], s[V];
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] = 0.f;
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            const int r = r0 + k * t.step + t.r;
            if (t.on && r < end) load_v<DT, V>(a.x, base + (int64_t)r * a.xt, f[k]);
            else {
#pragma unroll
                for (int e = 0; e < V; ++e) f[k][e] = 0.f;
            }
        }
#pragma unroll
        for (int k = 0; k < NR; ++k)
#pragma unroll
            for (int e = 0; e < V; ++e) s[e] += f[k][e];
        __syncthreads();
        put<V>(red, t, a.C, s);
        __syncthreads();
        group_sums(red, now, t, a.C, a.G, a.n, run);
        __syncthreads();
        const float rows = (float)min(end - r0, t.step * NR), inv = 1.f / (rows * (float)a.n);
        float mu[V];
#pragma unroll
        for (int e = 0; e < V; ++e) { mu[e] = t.on ? now[mine[e]] * inv : 0.f; s[e] = 0.f; }
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            if (r0 + k * t.step + t.r < end) {
#pragma unroll
                for (int e = 0; e < V; ++e) { const float d = f[k][e] - mu[e]; s[e] += d * d; }
            }
        }
        put<V>(red, t, a.C, s);
        // join with the tiles before: the mean first, while `now` still holds the sums
        const float share = rows / (before + rows);
        for (int g = threadIdx.x; g < a.G; g += blockDim.x) {
            const float d = now[g] * inv - mean[g];
            m2[g] += d * d * before * share * (float)a.n;
            mean[g] += d * share;
        }
        __syncthreads();
        group_sums(red, now, t, a.C, a.G, a.n, run);
        __syncthreads();
        for (int g = threadIdx.x; g < a.G; g += blockDim.x) m2[g] += now[g];
        before += rows;
    }
    __syncthreads();
    float2* out = reinterpret_cast<float2*>(a.part) + (int64_t)blockIdx.x * a.G;
    for (int g = threadIdx.x; g < a.G; g += blockDim.x) out[g] = make_float2(mean[g], m2[g]);
}

// joins the chunks' statistics (every workgroup for itself: a few hundred bytes), then normalises its chunk
template <int DT, int V, int NT>
__global__ __launch_bounds__(NT) void tile_apply_kernel(Args a) {
    extern __shared__ float lds[];
    float* mean = lds;
    float* rstd = lds + a.G;
    const Tile t(a.C, V);
    const int b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks, len = live_rows(a, b), run = run_of(a.chunks, 1, 1).lanes;
    const int first = chunk * a.rows_per_chunk, end = min(first + a.rows_per_chunk, a.T);
    const int per = blockDim.x / run, lane = threadIdx.x & (run - 1);
    const float2* part = reinterpret_cast<const float2*>(a.part) + (int64_t)b * a.chunks * a.G;
    const float inv = len > 0 ? 1.f / ((float)len * (float)a.n) : 0.f;
    for (int g0 = 0; g0 < a.G; g0 += per) {
        const int g = g0 + threadIdx.x / run;
        float2 p[MAX_CHUNKS / 64];
        float rows[MAX_CHUNKS / 64], mu = 0.f, var = 0.f;
#pragma unroll
        for (int i = 0; i < MAX_CHUNKS / 64; ++i) {
            const int k = lane + 64 * i;                   // (more than one where there are more than 64 chunks, whose run is 64 lanes)
            p[i] = make_float2(0.f, 0.f);
            rows[i] = g < a.G && k < a.chunks ? (float)min(max(len - k * a.rows_per_chunk, 0), a.rows_per_chunk) : 0.f;
            if (rows[i] > 0.f) p[i] = part[k * a.G + g];
            mu += p[i].x * (rows[i] * (float)a.n);
        }
        mu = lanes_sum(mu, run) * inv;
#pragma unroll
        for (int i = 0; i < MAX_CHUNKS / 64; ++i) { const float d = p[i].x - mu; var += p[i].y + d * d * (rows[i] * (float)a.n); }
        var = lanes_sum(var, run) * inv;
        if (g < a.G && lane == 0) {
            mean[g] = mu; rstd[g] = rsqrtf(var + a.eps);
            if (chunk == 0) { a.mean[(int64_t)b * a.G + g] = mean[g]; a.rstd[(int64_t)b * a.G + g] = rstd[g]; }
        }
    }
    __syncthreads();
    if (!t.on) return;
    float mu[V], w[V], bias[V];
    load_w<V>(a.w, t.v * V, 1.f, w);
    load_w<V>(a.bias, t.v * V, 0.f, bias);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = t.v * V + e, g = c / a.n;
        mu[e] = mean[g];
        w[e] *= rstd[g];
    }
    const int64_t xo = (int64_t)b * a.xb + t.v * V, oo = (int64_t)b * a.ob + t.v * V;
    int r = first + t.r;
    for (; r + 3 * t.step < min(end, len); r += 4 * t.step) {
        float f[4][V];
#pragma unroll
        for (int k = 0; k < 4; ++k) load_v<DT, V>(a.x, xo + (int64_t)(r + k * t.step) * a.xt, f[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
#pragma unroll
            for (int e = 0; e < V; ++e) f[k][e] = (f[k][e] - mu[e]) * w[e] + bias[e];
            activate<V>(f[k], a.act, a.slope);
            store_v<DT, V>(a.out, oo + (int64_t)(r + k * t.step) * a.ot, f[k]);
        }
    }
    for (; r < end; r += t.step) {
        float f[V];
        if (r < len) {
            load_v<DT, V>(a.x, xo + (int64_t)r * a.xt, f);
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = (f[e] - mu[e]) * w[e] + bias[e];
            activate<V>(f, a.act, a.slope);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = 0.f;
        }
        store_v<DT, V>(a.out, oo + (int64_t)r * a.ot, f);
    }
}

// sums of dz and dz xh of one chunk: part[(b * chunks + chunk) * 2 C + which * C + c]
template <int DT, int V, int NT>
__global__ __launch_bounds__(NT) void tile_dsum_kernel(Args a) {
    extern __shared__ float red[];
    constexpr int RU = NT > 256 && V > 4 ? 2 : 4;          // rows under way (four of them would not fit the registers that 1024 threads leave)
    const Tile t(a.C, V);
    const int b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks, len = live_rows(a, b);
    const int first = chunk * a.rows_per_chunk, end = min(first + a.rows_per_chunk, len);
    float s1[V], s2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s1[e] = s2[e] = 0.f;
    if (t.on) {
        float mu[V], rs[V], w[V], bias[V];
        load_w<V>(a.w, t.v * V, 1.f, w);
        load_w<V>(a.bias, t.v * V, 0.f, bias);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int c = t.v * V + e, g = c / a.n;
            mu[e] = a.mean[(int64_t)b * a.G + g]; rs[e] = a.rstd[(int64_t)b * a.G + g];
        }
        const int64_t xo = (int64_t)b * a.xb + t.v * V, po = (int64_t)b * a.db_ + t.v * V;
        for (int r0 = first + t.r; r0 < end; r0 += RU * t.step) {
            float f[RU][V], d[RU][V];
#pragma unroll
            for (int k = 0; k < RU; ++k) {
                const int r = r0 + k * t.step;
                if (r < end) { load_v<DT, V>(a.x, xo + (int64_t)r * a.xt, f[k]); load_v<DT, V>(a.dy, po + (int64_t)r * a.dt_, d[k]); }
                else {
#pragma unroll
                    for (int e = 0; e < V; ++e) f[k][e] = d[k][e] = 0.f;
                }
            }
#pragma unroll
            for (int k = 0; k < RU; ++k) {
                float z[V];
#pragma unroll
                for (int e = 0; e < V; ++e) { f[k][e] = (f[k][e] - mu[e]) * rs[e]; z[e] = f[k][e] * w[e] + bias[e]; }
                slopes<V>(z, a.act, a.slope);
#pragma unroll
                for (int e = 0; e < V; ++e) { const float dz = d[k][e] * z[e]; s1[e] += dz; s2[e] += r0 + k * t.step < end ? dz * f[k][e] : 0.f; }
            }
        }
    }
    float* out = a.part + (int64_t)blockIdx.x * 2 * a.C;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
        put<V>(red, t, a.C, which ? s2 : s1);
        __syncthreads();
        const Run run = run_of(1, a.C, t.step);
        group_sums(red, out + which * a.C, t, a.C, a.C, 1, run);
    }
}

// (items of per_item rows, 2, C) partial sums -> sums of each item.  A workgroup: 32 channels of one of the two sums, 32 items.
__global__ __launch_bounds__(1024) void item_kernel(const float* __restrict__ part, int items, int per_item, int C, float* __restrict__ item) {
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), which = blockIdx.y;
    const int64_t b = (int64_t)blockIdx.z * 32 + (threadIdx.x >> 5);
    if (c >= C || b >= items) return;
    const float* at = part + (b * per_item * 2 + which) * C + c;
    float t[4] = {};
    int k = 0;
    for (; k + 3 < per_item; k += 4)
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] += at[(int64_t)(k + i) * 2 * C];
    for (; k < per_item; ++k) t[0] += at[(int64_t)k * 2 * C];
    item[(b * 2 + which) * C + c] = (t[0] + t[1]) + (t[2] + t[3]);
}

// (rows, 2, C) -> sums over segments of `seg` rows, into out0 + segment * stride for [0] and out1 for [1] (null: not wanted).  A workgroup: 32 channels x 32 slots of
// rows, added in order.
__global__ __launch_bounds__(1024) void join_kernel(const float* __restrict__ part, int rows, int seg, int C, float* __restrict__ out0, float* __restrict__ out1, int64_t stride) {
    __shared__ float red[32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), slot = threadIdx.x >> 5, which = blockIdx.y;
    const int first = blockIdx.z * seg, end = min(rows, first + seg);
    float total = 0.f;
    if (c < C) {
        const float* at = part + (int64_t)which * C + c;
        float t[4] = {};
        int r = first + slot;
        for (; r + 96 < end; r += 128)
#pragma unroll
            for (int k = 0; k < 4; ++k) t[k] += at[(int64_t)(r + 32 * k) * 2 * C];
        for (; r < end; r += 32) t[0] += at[(int64_t)r * 2 * C];
        total = (t[0] + t[1]) + (t[2] + t[3]);
    }
    float* out = which ? out1 : out0;
    red[slot][threadIdx.x & 31] = total;
    __syncthreads();
    if (out && threadIdx.x < 32 && c < C) {
        float v = 0.f;
        for (int k = 0; k < 32; ++k) v += red[k][threadIdx.x];
        out[blockIdx.z * stride + c] = v;
    }
}

template <int DT, int V, int NT>
__global__ __launch_bounds__(NT) void tile_dx_kernel(Args a) {
    extern __shared__ float lds[];
    float* m1 = lds;                       // means of w dz and w dz xh of each group
    float* m2 = lds + a.G;
    const Tile t(a.C, V);
    const int b = blockIdx.x / a.chunks, chunk = blockIdx.x - b * a.chunks, len = live_rows(a, b), run = run_of(a.n, 1, 1).lanes;
    const int first = chunk * a.rows_per_chunk, end = min(first + a.rows_per_chunk, a.T);
    const int per = blockDim.x / run, lane = threadIdx.x & (run - 1);
    const float* item = a.item + (int64_t)b * 2 * a.C;
    const float inv = len > 0 ? 1.f / ((float)len * (float)a.n) : 0.f;
    for (int g0 = 0; g0 < a.G; g0 += per) {
        const int g = g0 + threadIdx.x / run;
        float v1 = 0.f, v2 = 0.f;
        if (g < a.G)
            for (int c = g * a.n + lane; c < (g + 1) * a.n; c += run) {
                const float w = a.w ? a.w[c] : 1.f;
                v1 += w * item[c]; v2 += w * item[a.C + c];
            }
        v1 = lanes_sum(v1, run); v2 = lanes_sum(v2, run);
        if (g < a.G && lane == 0) { m1[g] = v1 * inv; m2[g] = v2 * inv; }
    }
    __syncthreads();
    if (!t.on) return;
    float mu[V], rs[V], w[V], bias[V], k1[V], k2[V];
    load_w<V>(a.w, t.v * V, 1.f, w);
    load_w<V>(a.bias, t.v * V, 0.f, bias);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const int c = t.v * V + e, g = c / a.n;
        mu[e] = a.mean[(int64_t)b * a.G + g]; rs[e] = a.rstd[(int64_t)b * a.G + g];
        k1[e] = m1[g]; k2[e] = m2[g];
    }
    const int64_t xo = (int64_t)b * a.xb + t.v * V, po = (int64_t)b * a.db_ + t.v * V, oo = (int64_t)b * a.ob + t.v * V;
    for (int r0 = first + t.r; r0 < end; r0 += 2 * t.step) {
        float f[2][V], d[2][V];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int r = r0 + k * t.step;
            if (r < end && r < len) { load_v<DT, V>(a.x, xo + (int64_t)r * a.xt, f[k]); load_v<DT, V>(a.dy, po + (int64_t)r * a.dt_, d[k]); }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int r = r0 + k * t.step;
            if (r >= end) continue;
            if (r < len) {
                float z[V];
#pragma unroll
                for (int e = 0; e < V; ++e) { f[k][e] = (f[k][e] - mu[e]) * rs[e]; z[e] = f[k][e] * w[e] + bias[e]; }
                slopes<V>(z, a.act, a.slope);
#pragma unroll
                for (int e = 0; e < V; ++e) f[k][e] = rs[e] * (w[e] * (d[k][e] * z[e]) - k1[e] - f[k][e] * k2[e]);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) f[k][e] = 0.f;
            }
            store_v<DT, V>(a.out, oo + (int64_t)r * a.ot, f[k]);
        }
    }
}

// -------------------------------------------------------------------------------- plan ----
enum { SLAB, WHOLE, TILE };
struct Plan {
    int v;                                  // elements of a vector: 16 bytes, two or one
    int form, nv;                           // vectors of a thread: slab and whole forms
    SlabPlan s; int slab_wgs;
    WholePlan w; int whole_wgs;
    int threads, rows_per_chunk, chunks;
};

int pow2_at_least(int64_t x) { int r = 1; while (r < x) r <<= 1; return r; }

// widest of 16 bytes, two values and one that divides x and is allowed
int widest(int dtype, int allowed, int x) {
    const int wide = dtype == 0 ? 4 : 8;
    return allowed >= wide && x % wide == 0 ? wide : (allowed >= 2 && x % 2 == 0 ? 2 : 1);
}
// rows of dw / dbias partial sums that one workgroup of the join adds: beyond it, segments first
constexpr int JOIN_ROWS = 1024;
int join_segment(int64_t rows) { return (int)(rows <= (int64_t)JOIN_ROWS * JOIN_ROWS ? JOIN_ROWS : (rows + JOIN_ROWS - 1) / JOIN_ROWS); }
int join_segments(int64_t rows) { return (int)((rows + join_segment(rows) - 1) / join_segment(rows)); }

bool make_plan(const xva_group_norm_args* p, int vec, bool bwd, Plan* out) {
    Plan& q = *out;
    const int n = p->C / p->G;
    q.v = widest(p->dtype, vec, p->C);
    // slab form: a (item, group) slab of whole vectors within 64 lanes x 4 vectors (8 where they are narrow)
    const int sv = widest(p->dtype, vec, n);
    const int64_t vecs = (int64_t)p->T * (n / sv);
    if (vecs <= (sv <= 2 ? 512 : 256)) {
        q.form = SLAB;
        q.v = sv;
        q.nv = vecs <= 64 ? 1 : (vecs <= 128 ? 2 : (vecs <= 256 ? 4 : 8));
        q.s.lpg = pow2_at_least((vecs + q.nv - 1) / q.nv);
        const int slots = 256 / q.s.lpg;
        q.s.gpb = p->G < slots ? p->G : slots;
        q.s.ipb = slots / q.s.gpb;
        q.s.gy = (p->G + q.s.gpb - 1) / q.s.gpb;
        // several turns of items to a workgroup: its weights are loaded once, and one item's loads are under way while another is computed.  Eight workgroups to a
        // CU, four backward, where each leaves a partial row of dw / dbias.
        const int64_t want = ((int64_t)p->B + q.s.ipb - 1) / q.s.ipb;
        int64_t most = (bwd ? 1024 : 2048) / q.s.gy;
        if (most < 64) most = 64;
        q.slab_wgs = (int)(want < most ? want : most);
        return true;
    }
    // whole form: groups of one item within the registers of 512 threads (16 packed vectors to a thread, 12 of x and 12 of dy backward).  As many groups as make
    // 64 bytes of a row, more where workgroups abound.
    if (sv > 1) {
        const int nv = n / sv, cap = 512 * (bwd ? 12 : 16), line = 64 / (sv * xva_seq::elem_size(p->dtype));      // vectors of 64 bytes
        int gpw = (line + nv - 1) / nv;
        if (gpw > p->G) gpw = p->G;
        while (gpw > 1 && (int64_t)p->T * nv * gpw > cap) --gpw;
        while (gpw * 2 <= p->G && gpw * 2 * nv <= 4 * line && (int64_t)p->T * nv * gpw * 2 <= cap && (int64_t)p->B * ((p->G + 2 * gpw - 1) / (2 * gpw)) >= 512) gpw *= 2;
        const int lv = gpw * nv;
        if (lv <= 512 && (int64_t)p->T * nv * gpw <= (int64_t)(512 / lv) * lv * (bwd ? 12 : 16)) {
            q.form = WHOLE;
            q.w.gpw = gpw; q.w.lv = lv;
            q.w.threads = (int64_t)p->T * lv <= 4 * 256 && lv <= 256 ? 256 : 512;
            q.w.rows = q.w.threads / lv;
            q.w.blocks = (p->G + gpw - 1) / gpw;
            const int each = (p->T + q.w.rows - 1) / q.w.rows;
            q.nv = each <= 4 ? 4 : (each <= 8 ? 8 : (each <= 12 ? 12 : 16));
            q.whole_wgs = (int)(((int64_t)p->B * q.w.blocks + 7) / 8 * 8);
            if (each <= (bwd ? 12 : 16)) { q.v = sv; return true; }
        }
    }
    q.form = TILE;
    const int lc = p->C / q.v;
    if (lc > 1024 || p->G > 2048) return false;        // (a row in one workgroup, its groups in the LDS)
    q.threads = lc <= 256 ? 256 : (lc + 63) / 64 * 64;
    const int step = q.threads / lc;
    // chunks of whole register tiles where there are rows for four workgroups to a CU, of fewer rows where there are not; at most 256 of an item (four to a
    // lane when they are joined)
    int64_t turns = (p->T + step - 1) / step, want = (1024 + p->B - 1) / p->B;
    if (want > MAX_CHUNKS) want = MAX_CHUNKS;
    if (want > turns) want = turns;
    int64_t each = (turns + want - 1) / want;
    if (each > NR) each = (each + NR - 1) / NR * NR;
    q.rows_per_chunk = (int)(each * step);
    q.chunks = (int)((p->T + q.rows_per_chunk - 1) / q.rows_per_chunk);
    return true;
}

// the widest vector that strides and addresses allow
int allowed(const xva_group_norm_args* p, bool bwd) {
    const int wide = p->dtype == 0 ? 4 : 8;
    int64_t all = p->x_stride[0] | p->x_stride[1] | p->out_stride[0] | p->out_stride[1];
    uintptr_t ptrs = (uintptr_t)p->x | (uintptr_t)p->out;
    if (bwd) { all |= p->dy_stride[0] | p->dy_stride[1]; ptrs |= (uintptr_t)p->dy; }
    if (all % wide == 0 && ptrs % 16 == 0) return wide;
    return all % 2 == 0 && ptrs % (2 * xva_seq::elem_size(p->dtype)) == 0 ? 2 : 1;
}

int check(const xva_group_norm_args* p, const char* who) {
    XVA_CHECK_ARG(p, "%s: null argument", who);
    XVA_CHECK_ARG(p->dtype >= 0 && p->dtype <= 2, "%s: dtype %d", who, p->dtype);
    XVA_CHECK_ARG(p->B >= 0 && p->B < (1 << 30) && p->T >= 0 && p->T < (1 << 30) && p->C >= 1 && p->C <= 65536 && p->G >= 1 && p->C % p->G == 0, "%s: B %d T %d C %d in %d groups", who, p->B, p->T, p->C, p->G);
    XVA_CHECK_ARG(p->act >= NONE && p->act <= GELU, "%s: activation %d", who, p->act);
    XVA_CHECK_ARG(p->eps >= 0.f, "%s: eps %g", who, p->eps);
    XVA_CHECK_ARG(p->B == 0 || p->T == 0 || (p->x && p->out && p->mean && p->rstd), "%s: null argument", who);
    return XVA_OK;
}

Args args_of(const xva_group_norm_args* p, const Plan& q) {
    Args a = {};
    a.x = p->x; a.dy = p->dy; a.out = p->out; a.w = p->weight; a.bias = p->bias; a.lens = p->lens; a.mean = p->mean; a.rstd = p->rstd;
    a.dw = p->dweight; a.db = p->dbias;
    a.xb = p->x_stride[0]; a.xt = p->x_stride[1]; a.ob = p->out_stride[0]; a.ot = p->out_stride[1]; a.db_ = p->dy_stride[0]; a.dt_ = p->dy_stride[1];
    a.B = p->B; a.T = p->T; a.C = p->C; a.G = p->G; a.n = p->C / p->G; a.act = p->act; a.eps = p->eps; a.slope = p->slope;
    a.rows_per_chunk = q.rows_per_chunk; a.chunks = q.chunks;
    return a;
}

int64_t workspace(const xva_group_norm_args* p, bool bwd) {
    if (p->B == 0 || p->T == 0) return 0;
    // (over the vector widths: which one runs depends on addresses and strides)
    int64_t most = 0;
    for (int vec = 8; vec > 0; vec = vec == 8 ? 2 : vec - 1) {
        Plan q = {};
        if (!make_plan(p, vec, bwd, &q)) continue;
        int64_t f;
        if (q.form == TILE) f = bwd ? (int64_t)p->B * (q.chunks + (q.chunks > 1)) * 2 * p->C : (int64_t)p->B * q.chunks * 2 * p->G;
        else f = bwd ? (q.form == SLAB ? (int64_t)q.slab_wgs : (int64_t)p->B) * 2 * p->C : 0;
        if (bwd) f += (int64_t)join_segments(q.form == SLAB ? q.slab_wgs : p->B) * 2 * p->C;
        if (f > most) most = f;
    }
    return most * 4;
}

template <int DT, int V, bool BWD> int slab_launch(const Args& a, const Plan& q, hipStream_t st) {
    const dim3 grid(q.slab_wgs, q.s.gy);
    const size_t lds = BWD ? (size_t)256 * q.nv * 2 * V * 4 : 0;
    if (q.nv == 1) slab_kernel<DT, V, 1, BWD><<<grid, 256, lds, st>>>(a, q.s);
    else if (q.nv == 2) slab_kernel<DT, V, 2, BWD><<<grid, 256, lds, st>>>(a, q.s);
    else if (q.nv == 4) slab_kernel<DT, V, 4, BWD><<<grid, 256, lds, st>>>(a, q.s);
    else if constexpr (V <= 2) slab_kernel<DT, V, 8, BWD><<<grid, 256, lds, st>>>(a, q.s);
    XVA_LAUNCH_CHECK();
    return XVA_OK;
}

template <int DT, int V, bool BWD> int whole_launch(const Args& a, const Plan& q, hipStream_t st) {
    if constexpr (V == 1) { return XVA_ERR_ARG; }
    else {
        const int cw = q.w.lv * V;
        const size_t lds = (BWD ? (size_t)q.w.rows * cw + 2 * cw : (size_t)q.w.threads) * 4 + 2 * q.w.gpw * 4;
        const dim3 grid(q.whole_wgs);
        switch (q.nv) {
            case 4: whole_kernel<DT, V, 4, BWD><<<grid, q.w.threads, lds, st>>>(a, q.w); break;
            case 8: whole_kernel<DT, V, 8, BWD><<<grid, q.w.threads, lds, st>>>(a, q.w); break;
            case 12: whole_kernel<DT, V, 12, BWD><<<grid, q.w.threads, lds, st>>>(a, q.w); break;
            default: if constexpr (!BWD) whole_kernel<DT, V, 16, BWD><<<grid, q.w.threads, lds, st>>>(a, q.w);
        }
        XVA_LAUNCH_CHECK();
        return XVA_OK;
    }
}

template <int DT, int V> int forward(Args& a, const Plan& q, hipStream_t st) {
    if (q.form == WHOLE) return whole_launch<DT, V, false>(a, q, st);
    if (q.form == SLAB) return slab_launch<DT, V, false>(a, q, st);
    const dim3 grid((unsigned)(a.B * q.chunks));
    const int step = q.threads / (a.C / V);
    if (q.threads <= 256) tile_stats_kernel<DT, V, 256><<<grid, q.threads, ((size_t)step * a.C + 3 * a.G) * 4, st>>>(a);
    else tile_stats_kernel<DT, V, 1024><<<grid, q.threads, ((size_t)step * a.C + 3 * a.G) * 4, st>>>(a);
    XVA_LAUNCH_CHECK();
    if (q.threads <= 256) tile_apply_kernel<DT, V, 256><<<grid, q.threads, (size_t)2 * a.G * 4, st>>>(a);
    else tile_apply_kernel<DT, V, 1024><<<grid, q.threads, (size_t)2 * a.G * 4, st>>>(a);
    XVA_LAUNCH_CHECK();
    return XVA_OK;
}

// dw, dbias from (rows, 2, C) partial sums; `spare` holds the segments' sums where there are several
int join(const Args& a, const float* part, int rows, float* spare, hipStream_t st) {
    if (!a.dw && !a.db) return XVA_OK;
    const int segs = join_segments(rows);
    if (segs > 1) {
        join_kernel<<<dim3((a.C + 31) / 32, 2, segs), 1024, 0, st>>>(part, rows, join_segment(rows), a.C, spare, spare + a.C, 2 * (int64_t)a.C);
        XVA_LAUNCH_CHECK();
        part = spare; rows = segs;
    }
    join_kernel<<<dim3((a.C + 31) / 32, 2), 1024, 0, st>>>(part, rows, rows, a.C, a.db, a.dw, 0);
    XVA_LAUNCH_CHECK();
    return XVA_OK;
}

template <int DT, int V> int backward(Args& a, const Plan& q, hipStream_t st) {
    if (q.form != TILE) {
        const int rows = q.form == SLAB ? q.slab_wgs : a.B;
        if (q.form == WHOLE) XVA_TRY((whole_launch<DT, V, true>(a, q, st)));
        else XVA_TRY((slab_launch<DT, V, true>(a, q, st)));
        return join(a, a.part, rows, a.part + (int64_t)rows * 2 * a.C, st);
    }
    const dim3 grid((unsigned)(a.B * q.chunks));
    const int step = q.threads / (a.C / V);
    const int64_t parts = (int64_t)a.B * q.chunks * 2 * a.C;
    a.item = q.chunks > 1 ? a.part + parts : a.part;
    if (q.threads <= 256) tile_dsum_kernel<DT, V, 256><<<grid, q.threads, (size_t)step * a.C * 4, st>>>(a);
    else tile_dsum_kernel<DT, V, 1024><<<grid, q.threads, (size_t)step * a.C * 4, st>>>(a);
    XVA_LAUNCH_CHECK();
    if (q.chunks > 1) {
        item_kernel<<<dim3((a.C + 31) / 32, 2, (a.B + 31) / 32), 1024, 0, st>>>(a.part, a.B, q.chunks, a.C, a.item);
        XVA_LAUNCH_CHECK();
    }
    if (q.threads <= 256) tile_dx_kernel<DT, V, 256><<<grid, q.threads, (size_t)2 * a.G * 4, st>>>(a);
    else tile_dx_kernel<DT, V, 1024><<<grid, q.threads, (size_t)2 * a.G * 4, st>>>(a);
    XVA_LAUNCH_CHECK();
    return join(a, a.item, a.B, a.item + (int64_t)a.B * 2 * a.C, st);
}

int run(const xva_group_norm_args* p, bool bwd, void* ws, int64_t ws_bytes, void* stream, const char* who) {
    XVA_TRY(check(p, who));
    XVA_CHECK_ARG(!bwd || p->dy || p->B == 0 || p->T == 0, "%s: null gradient", who);
    hipStream_t st = (hipStream_t)stream;
    // (before any plan: it divides the workgroups among the items)
    if (p->B == 0 || p->T == 0) {
        if (bwd) {
            if (p->dweight) { void* d[1] = {p->dweight}; const int64_t n[1] = {(int64_t)p->C * 4}; XVA_TRY(xva_zero_spans(d, n, 1, stream)); }
            if (p->dbias) { void* d[1] = {p->dbias}; const int64_t n[1] = {(int64_t)p->C * 4}; XVA_TRY(xva_zero_spans(d, n, 1, stream)); }
        }
        return XVA_OK;
    }
    Plan q = {};
    // (the forward refuses what the backward would have to)
    XVA_CHECK_ARG((bwd || make_plan(p, allowed(p, false), true, &q)) && make_plan(p, allowed(p, bwd), bwd, &q), "%s: %d channels in %d groups: at most 2048 groups and 1024 vectors of %d channels", who, p->C, p->G, q.v);
    XVA_CHECK_ARG(q.form == SLAB || xva_seq::launchable((int64_t)p->B * (q.form == TILE ? q.chunks : q.w.blocks) + 7, q.form == TILE ? q.threads : q.w.threads),
                  "%s: %d items of %d rows", who, p->B, p->T);
    const int64_t need = workspace(p, bwd);
    if (ws_bytes < need || (need && !ws)) { xva_set_error("%s: workspace of %lld bytes, %lld needed", who, (long long)ws_bytes, (long long)need); return XVA_ERR_WS; }
    Args a = args_of(p, q);
    a.part = (float*)ws;
#define GN(DT, V) (bwd ? backward<DT, V>(a, q, st) : forward<DT, V>(a, q, st))
#define GNV(DT, WIDE) return q.v == WIDE ? GN(DT, WIDE) : (q.v == 2 ? GN(DT, 2) : GN(DT, 1))
    if (p->dtype == 0) GNV(0, 4);
    if (p->dtype == 1) GNV(1, 8);
    GNV(2, 8);
#undef GNV
#undef GN
}
}   // namespace

extern "C" int64_t xva_group_norm_workspace_bytes(const xva_group_norm_args* p, int backward_pass) {
    if (!p || p->G < 1 || p->C < 1 || p->C % p->G || p->B < 0 || p->T < 0 || p->T >= (1 << 30)) return -1;
    return workspace(p, backward_pass != 0);
}
extern "C" int xva_group_norm_act_fwd(const xva_group_norm_args* p, void* ws, int64_t ws_bytes, void* stream) {
    return run(p, false, ws, ws_bytes, stream, "xva_group_norm_act_fwd");
}
extern "C" int xva_group_norm_act_bwd(const xva_group_norm_args* p, void* ws, int64_t ws_bytes, void* stream) {
    return run(p, true, ws, ws_bytes, stream, "xva_group_norm_act_bwd");
}
