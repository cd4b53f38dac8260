// rotary.hip — rotary positions on the query and key heads of a sequence (gfx950).
//
// Pair (a, b) of a head at position p turns by the angle p w:   a' = m (a cos - b sin),  b' = m (b cos + a sin),   w = the pair's frequency, m = the plan's gain.
// The gradient is the same map with the angle negated, so forward and backward are one kernel.
//
// Bound: HBM — one read and one write of q and k.  The angles are not read from a table over positions (at 128 of head width that is a fp32 table row of
// 512 bytes per token) but made on the spot, once per (token, pair), and shared by all heads through LDS: a workgroup owns a few tokens, first fills
// (cos, sin) of its tokens, then streams the tokens' heads in memory order.  bf16, 2 x 16384 tokens of 16 + 4 heads of 128: 336 MB in 65 - 70 us (5 TB/s, what a large
// copy reaches); 64 tokens of 16 + 4 heads of 96 (interleaved): 3.7 us, a launch.
//
// Angles of far positions: p w in fp32 is off by p w 2^-24 radians (half a radian at a position of 8 million).  The plan holds w / 2 pi as a 64-bit
// fixed-point fraction of a turn, so that p * w modulo one turn is the low half of an integer product: exact for every 64-bit position but for the table's
// own rounding (half a unit: p 2^-65 turns, fp32's own step at about 2^40).  sincospif then takes the reduced turn.
#include "xva_common.h"
#include "../../include/xva_hip.h"
#include "seq_vec.h"

namespace {
using xva_seq::load_v;
using xva_seq::store_v;

constexpr int THREADS = 256;
constexpr int LDS_PAIRS = 4096;       // (cos, sin) pairs of one workgroup: 32 KiB
constexpr int MAX_TOKENS = 16;        // tokens of one workgroup

struct Side { const void* x; void* y; int64_t xb, xt, xh, yb, yt, yh; int heads; };

struct Args {
    Side s[2];                        // queries, keys
    const uint64_t* turns;            // rd / 2 fractions of a turn per position, 64-bit fixed point
    const void* pos; int pos64; int64_t pb, pt;   // positions (null: the row's index)
    float gain, sign;
    int B, T, D, rd, per_wg;
};

// A work item is V pairs of one (token, head), or 2 V elements of its part that does not turn.  Items of a row lie side by side over the lanes.
// V = 0: one pair, element by element (any alignment), or one element of the still part; V = 1 in the half layout takes any alignment as it is.
template <int DT, bool INTER, int V>
__global__ __launch_bounds__(THREADS) void rotary_kernel(Args a) {
    extern __shared__ float2 cs[];         // (cos, sin) of the workgroup's tokens
    __shared__ int64_t at[MAX_TOKENS][4];  // where each token's heads start: queries in and out, keys in and out
    constexpr int P = V ? V : 1;           // pairs of an item
    constexpr bool ONE = INTER ? V == 0 : V == 1;      // elements one by one
    const int np = a.rd >> 1;
    const unsigned tok0 = blockIdx.x * (unsigned)a.per_wg;
    const int ntok = (int)min((unsigned)a.per_wg, (unsigned)a.B * (unsigned)a.T - tok0);
    for (int e = threadIdx.x; e < ntok * np; e += THREADS) {
        const int tl = (unsigned)e / (unsigned)np, i = e - tl * np;
        const unsigned tok = tok0 + tl;
        const int b = (int)(tok / (unsigned)a.T), t = (int)(tok - (unsigned)b * (unsigned)a.T);
        if (i == 0) {
#pragma unroll
            for (int k = 0; k < 2; ++k) { at[tl][2 * k] = b * a.s[k].xb + t * a.s[k].xt; at[tl][2 * k + 1] = b * a.s[k].yb + t * a.s[k].yt; }
        }
        int64_t p = t;
        if (a.pos) {
            const int64_t where = b * a.pb + t * a.pt;
            p = a.pos64 ? reinterpret_cast<const int64_t*>(a.pos)[where] : (int64_t)reinterpret_cast<const int32_t*>(a.pos)[where];
        }
        const float turn = (float)(int64_t)((uint64_t)p * a.turns[i]);      // in units of 2^-64 turns, -2^63 .. 2^63: within half a turn of zero
        float sn, c;
        sincospif(turn * 0x1p-63f, &sn, &c);
        cs[e] = make_float2(c * a.gain, sn * a.gain * a.sign);
    }
    __syncthreads();
    const int HT = a.s[0].heads + a.s[1].heads;
    // (in place the part that does not turn stays where it is)
    const int turning = np / P, still = (a.s[0].x == a.s[0].y) ? 0 : (ONE ? a.D - a.rd : (a.D - a.rd) / (2 * P));
    const int per_row = turning + still;
    const int lanes = min(per_row, THREADS), rows_at_once = THREADS / lanes;
    const int lane = threadIdx.x % lanes, first = threadIdx.x / lanes;
    if (first >= rows_at_once) return;
    const int step_t = rows_at_once / HT, step_h = rows_at_once - step_t * HT;
    int tl = first / HT, h = first - tl * HT;
    while (tl < ntok) {
        const bool key = h >= a.s[0].heads;
        const uint32_t hh = key ? h - a.s[0].heads : h;
        const void* x = key ? a.s[1].x : a.s[0].x;
        void* y = key ? a.s[1].y : a.s[0].y;
        const int64_t xo = at[tl][key ? 2 : 0] + (int64_t)((uint64_t)hh * (key ? a.s[1].xh : a.s[0].xh)), yo = at[tl][key ? 3 : 1] + (int64_t)((uint64_t)hh * (key ? a.s[1].yh : a.s[0].yh));
        for (int c = lane; c < per_row; c += lanes) {
            if (c < turning) {
                const float2* w = cs + tl * np + c * P;
                if constexpr (INTER) {
                    float f[2 * P];
                    if constexpr (ONE) {
                        float u[1];
                        load_v<DT, 1>(x, xo + 2 * c, u); f[0] = u[0];
                        load_v<DT, 1>(x, xo + 2 * c + 1, u); f[1] = u[0];
                    } else load_v<DT, 2 * P>(x, xo + 2 * P * c, f);
#pragma unroll
                    for (int e = 0; e < P; ++e) {
                        const float2 k = w[e];
                        const float u = f[2 * e] * k.x - f[2 * e + 1] * k.y, v = f[2 * e + 1] * k.x + f[2 * e] * k.y;
                        f[2 * e] = u; f[2 * e + 1] = v;
                    }
                    if constexpr (ONE) {
                        const float u[1] = {f[0]}, v[1] = {f[1]};
                        store_v<DT, 1>(y, yo + 2 * c, u); store_v<DT, 1>(y, yo + 2 * c + 1, v);
                    } else store_v<DT, 2 * P>(y, yo + 2 * P * c, f);
                } else {
                    float f[P], g[P];
                    load_v<DT, P>(x, xo + P * c, f);
                    load_v<DT, P>(x, xo + np + P * c, g);
#pragma unroll
                    for (int e = 0; e < P; ++e) {
                        const float2 k = w[e];
                        const float u = f[e] * k.x - g[e] * k.y, v = g[e] * k.x + f[e] * k.y;
                        f[e] = u; g[e] = v;
                    }
                    store_v<DT, P>(y, yo + P * c, f);
                    store_v<DT, P>(y, yo + np + P * c, g);
                }
            } else {
                constexpr int W = ONE ? 1 : 2 * P;
                float f[W];
                load_v<DT, W>(x, xo + a.rd + W * (c - turning), f);
                store_v<DT, W>(y, yo + a.rd + W * (c - turning), f);
            }
        }
        tl += step_t; h += step_h;
        if (h >= HT) { h -= HT; ++tl; }
    }
}

template <int DT, bool INTER> int launch(const Args& a, int v, dim3 grid, size_t lds, hipStream_t st) {
    switch (v) {
        case 8: if constexpr (DT != 0 && !INTER) { rotary_kernel<DT, INTER, 8><<<grid, THREADS, lds, st>>>(a); break; }
        case 4: rotary_kernel<DT, INTER, 4><<<grid, THREADS, lds, st>>>(a); break;
        case 2: rotary_kernel<DT, INTER, 2><<<grid, THREADS, lds, st>>>(a); break;
        case 1: rotary_kernel<DT, INTER, 1><<<grid, THREADS, lds, st>>>(a); break;
        default: rotary_kernel<DT, INTER, INTER ? 0 : 1><<<grid, THREADS, lds, st>>>(a);
    }
    XVA_LAUNCH_CHECK();
    return XVA_OK;
}
}   // namespace

extern "C" int xva_rotary(const xva_rotary_args* p, void* stream) {
    XVA_CHECK_ARG(p && p->turns, "xva_rotary: null argument");
    XVA_CHECK_ARG(p->dtype >= 0 && p->dtype <= 2, "xva_rotary: dtype %d", p->dtype);
    XVA_CHECK_ARG(p->B >= 0 && p->T >= 0 && p->H >= 1 && p->Hk >= 0 && p->Hk <= 65536 && p->H <= 65536, "xva_rotary: B %d T %d H %d Hk %d", p->B, p->T, p->H, p->Hk);
    XVA_CHECK_ARG(p->rd >= 2 && (p->rd & 1) == 0 && p->rd <= p->D && p->D <= 8192, "xva_rotary: rotary width %d of a head of %d", p->rd, p->D);
    if (p->B == 0 || p->T == 0) return XVA_OK;
    XVA_CHECK_ARG(p->q && p->q_out, "xva_rotary: null argument");
    XVA_CHECK_ARG(p->Hk == 0 || (p->k && p->k_out), "xva_rotary: null keys");
    XVA_CHECK_ARG(p->Hk == 0 || (p->q == p->q_out) == (p->k == p->k_out), "xva_rotary: queries and keys are both turned in place or both not");
    XVA_CHECK_ARG(p->q != p->q_out || (memcmp(p->q_stride, p->q_out_stride, sizeof p->q_stride) == 0 &&
                                       (p->Hk == 0 || memcmp(p->k_stride, p->k_out_stride, sizeof p->k_stride) == 0)), "xva_rotary: in place with other strides");
    Args a = {};
    a.s[0] = {p->q, p->q_out, p->q_stride[0], p->q_stride[1], p->q_stride[2], p->q_out_stride[0], p->q_out_stride[1], p->q_out_stride[2], p->H};
    a.s[1] = {p->k, p->k_out, p->k_stride[0], p->k_stride[1], p->k_stride[2], p->k_out_stride[0], p->k_out_stride[1], p->k_out_stride[2], p->Hk};
    a.turns = p->turns; a.pos = p->positions; a.pos64 = p->positions64; a.pb = p->pos_stride[0]; a.pt = p->pos_stride[1];
    a.gain = p->gain; a.sign = p->inverse ? -1.f : 1.f;
    a.B = p->B; a.T = p->T; a.D = p->D; a.rd = p->rd;
    // widest vector that divides both halves (half layout) / the pairs (interleaved), the still part and every stride and address
    const int es = p->dtype == 0 ? 4 : 2, np = p->rd / 2;
    int v = p->dtype != 0 && !p->interleaved ? 8 : 4;
    for (; v > (p->interleaved ? 0 : 1); v >>= 1) {
        const int el = p->interleaved ? 2 * v : v;                  // elements of one access, or 16 bytes where that is less
        const int al = el * es < 16 ? el : 16 / es;
        bool ok = np % v == 0 && (p->D - p->rd) % (2 * v) == 0;
        // the still part's accesses are 2 v wide and start at rd = 2 np, a multiple of 2 v
        const int al2 = 2 * v * es < 16 ? 2 * v : 16 / es, need = p->D > p->rd ? (al2 > al ? al2 : al) : al;
        for (int side = 0; side < (p->Hk ? 2 : 1); ++side) {
            const Side& s = a.s[side];
            const int64_t all = s.xb | s.xt | s.xh | s.yb | s.yt | s.yh | (int64_t)((uintptr_t)s.x / es) | (int64_t)((uintptr_t)s.y / es);
            ok = ok && all % need == 0;
        }
        if (ok) break;
    }
    // tokens per workgroup: enough workgroups to fill 256 CUs eight times before a workgroup takes a second token; (cos, sin) of all of them fit the LDS
    const int64_t tokens = (int64_t)p->B * p->T;
    XVA_CHECK_ARG(np <= LDS_PAIRS, "xva_rotary: rotary width %d", p->rd);
    XVA_CHECK_ARG(tokens < (1ll << 31), "xva_rotary: %lld tokens", (long long)tokens);
    int64_t per = tokens / 2048;
    if (per > MAX_TOKENS) per = MAX_TOKENS;
    if (per > LDS_PAIRS / np) per = LDS_PAIRS / np;
    if (per < 1) per = 1;
    const int64_t wgs = (tokens + per - 1) / per;
    XVA_CHECK_ARG(xva_seq::launchable(wgs, THREADS), "xva_rotary: %lld tokens, %lld to a workgroup", (long long)tokens, (long long)per);
    a.per_wg = (int)per;
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)wgs);
    const size_t lds = (size_t)per * np * sizeof(float2);
    if (p->interleaved) {
        if (p->dtype == 0) return launch<0, true>(a, v, grid, lds, st);
        return p->dtype == 1 ? launch<1, true>(a, v, grid, lds, st) : launch<2, true>(a, v, grid, lds, st);
    }
    if (p->dtype == 0) return launch<0, false>(a, v, grid, lds, st);
    return p->dtype == 1 ? launch<1, false>(a, v, grid, lds, st) : launch<2, false>(a, v, grid, lds, st);
}
