// diff_attention.hip — differential attention: the difference of two softmax maps over shared values, 16-bit operands (gfx950).
//
//   S_m = scale q_m k_m^T (m = 1, 2),  P_m = softmax(S_m) over the visible keys,  O = (P_1 - lam P_2) V,  lam a learned number of each head
//   dP = dO V^T,  D_m = rowsum(dO o P_m V),  dS_1 = P_1 o (dP - D_1),  dS_2 = -lam P_2 o (dP - D_2)
//   dq_m = scale dS_m k_m,  dk_m = scale dS_m^T q_m,  dV = (P_1 - lam P_2)^T dO,  dlam = - sum P_2 o dP
//   Key heads may be fewer than query heads (their gradients add up); a query of an item with ql queries and kl keys sees keys j < kl, and with `causal`
//   j <= i + kl - ql.  A row that sees nothing leaves as zeros and gives no gradient.
//
// Bound: MFMA and the exponentials beside it.  No score leaves the chip.
//   forward : a workgroup takes 128 queries of a head (64 of the narrower ones), 32 to a wave; the two maps run their own online softmax over 64-key tiles and share every fragment of
//             V (one LDS read feeds both maps' products).  Base-2 exponentials, the scale folded in; the running maximum is only moved when a tile exceeds it
//             by 2^8, so the accumulators are rescaled in the first tiles and hardly ever after.
//   backward: dK / dV by key block and dq by query block, each rebuilding the maps from the saved logsumexp; no atomics, so results repeat bit for bit.
//             dP is shared by both maps, and dV takes P_1 - lam P_2 in one product: 16 d + 12 d multiply-adds x 2 a pair and head (d: width of one map's
//             query).  dlam is summed from fp32 P_2 o dP beside dq, not from rounded outputs.
// Waves raise their priority over the products that follow a softmax (s_setprio): the other wave of a SIMD then does its exponentials meanwhile (8192 causal positions,
// heads of 64: dq 463 -> 429 us, dK/dV 692 -> 673, forward 484 -> 476; over the score products as well: 481, 699, 474).
// Reached (kernels' time, dense operations of the formulas): 8192 causal positions, 16 heads of 64 on 4 keys' 472 us forward (870 TFLOP/s), 1070 us dK / dV / dq (640):
// CUs busy 86 and 93 % of the launch, while they are matrix units 47 and 46 %, vector units 59 and 56 %, two waves to a SIMD, at 2.0 GHz.  32 x 860 ragged frames, fp16,
// 4 heads of 48: 82 + 158 us: 688 query blocks on 512 places, and scores of 48 columns take matrix steps of 64.  32 x 150, heads of 32: 13 + 16 us and 9 for the two
// small launches, each a chain of latencies.  One query on each of 16 ragged caches of up to 8192 keys, 16 heads of 64 on 4 keys': 41 us (4.7 TB/s) and 7 for the join.
// Roundings: P, P_1 - lam P_2 and dS to the tensors' 16-bit type as MFMA operands, which is what the matrix units take at this rate; each map's own output, to the
// tensors' type, kept for the backward pass, whose D_m is made from it (in fp32 it would be another 2 x 4 bytes a value, written and read).  Accumulators, scores, sums,
// maxima, logsumexp and D stay fp32.  fp16 holds dS by powers of two in its normal range (range_kernel).
//
// Tiles: 64 rows x 64 columns of 16-bit values (attn_tile.h).  d <= 32: one image holds both maps' 32 columns side by side; d <= 64: one image for each map.
// V and dO (2 d wide): one or two images.  Rows behind the last live one read that one, with P = 0.
#include "attn_tile.h"
#include "../../include/xva_hip.h"
#include "seq_vec.h"

namespace {
using namespace xva_glds;
using xva_attn::Frag;
using xva_attn::TILE;
using xva_attn::pack_rows;

struct Args {
    const uint16_t *q, *k, *v, *dout;
    uint16_t *out, *maps, *dq, *dk, *dv;
    const void* lam;                              // (H) of type lam_type: 0 fp32, 1 bf16, 2 fp16
    int lam_type;
    float* lam32;                                 // backward: the same in fp32, for the scalar unit (rowdot_kernel leaves it)
    float *lse, *D, *dlam_part;
    float *norms;                                 // fp16 backward: largest squared norm of each 16 rows of dO (B, H, Tq / 16), then of v (B, Hk, Tk / 16)
    float *start;                                 // fp16 backward: lse and D as dkv takes them (range_kernel)
    float *range;                                 // fp16 backward: of each (item, key head) the factors that keep dS in the type's range (see range_kernel)
    const int32_t *ql, *kl;
    int64_t qb, qt, qh, qm, kb, kt, kh, km, vb, vt, vh, ob, ot, oh, gb, gt, gh;
    int B, Tq, Tk, H, Hk, share, d, causal;
    float scale, c;                               // c = scale log2 e
    // dkv: workgroups of a key block, and the tiles that one of them takes; forward and dq: the same of a query block (see dkv_kernel)
    float* part; int pieces, piece;
    float* qpart; int qpieces, qpiece;
};
// contiguous results: out-of-line maps (2, B, Tq, H, 2 d), dq (B, Tq, H, 2, d), dk (B, Tk, Hk, 2, d), dv (B, Tk, Hk, 2 d)
// lse (2, B, H, Tq): minus the row's logarithm of sums, in units of unscaled scores (-inf: the row sees nothing), so P = exp2(c (S + lse)); D (2, B, H, Tq): -D_1
// and D_1 - D_2.  Both are what dkv's matrix products start from.

template <int D16> struct Shape {
    static constexpr int NI = D16 <= 2 ? 1 : 2;   // 64-column images of a q / k tile, and of a v / dO tile
    static constexpr int KH = NI;                 // 32-wide MFMA steps over d of one map
    static constexpr int VH = NI * 2;             // 32-wide MFMA steps over 2 d
    static constexpr int DT = D16;                // 16-column tiles of one map's d
    static constexpr int VT = D16 * 2;            // 16-column tiles of 2 d
};

__device__ __forceinline__ int len_of(const int32_t* l, int b, int T) { return l ? min(max(l[b], 0), T) : T; }

// 16 bytes to LDS from `rows` + `off` bytes, within the `bytes` that are there.  A buffer load: the compiler counts it like any load, where the global form's wait
// would be for everything in flight.
__device__ __forceinline__ void load_lds(const uint16_t* rows, uint32_t bytes, uint32_t off, XVA_LDS uint8_t* to) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void*)rows, 0, bytes, 0x00027000), (XVA_LDS void*)to, 16, off, 0, 0, 0);
}
// Where this lane's two 16-byte pieces of an image come from: rows r and r + 32 of the tile, one column (the swizzle repeats every 8 rows).  Columns behind the
// width read the row's first ones: they meet zeros in the other operand, or results that nobody stores, and a row that is not finite is lost through its
// live columns already.
template <int NI> struct Src {
    uint32_t r, qk[NI], v[NI];                    // row, and the column's byte offset in each image: a q / k tile's (one image: with the map's), a v / dO tile's
    __device__ __forceinline__ Src(int lane, int wave, int d, int64_t map_stride) {
        r = wave * 8 + (lane >> 3);
        const int p = lane & 7, c = (((p >> 1) ^ ((r >> 1) & 3)) << 1) | (p & 1);
#pragma unroll
        for (int im = 0; im < NI; ++im) {
            const int d0 = (NI == 2 ? c : c & 3) * 8, e0 = im * 64 + c * 8;
            qk[im] = 2u * ((NI == 2 ? 0u : (uint32_t)(c >> 2) * (uint32_t)map_stride) + (d0 < d ? d0 : 0));
            v[im] = 2u * (e0 < 2 * d ? e0 : 0);
        }
    }
    // the `left` (>= 1) rows from `rows` on, clamped to the last of them; images `apart` elements from each other, `width` elements behind a row's first one
    __device__ __forceinline__ void fetch(const uint16_t* rows, int64_t ld, int64_t apart, int64_t width, const uint32_t (&col)[NI], int left, XVA_LDS uint8_t* tile, int wave) const {
        const uint32_t ldb = (uint32_t)ld * 2u, bytes = (uint32_t)(min(left, 64) - 1) * ldb + (uint32_t)width * 2u;
        const uint32_t at[2] = {min(r, (uint32_t)left - 1) * ldb, min(r + 32, (uint32_t)left - 1) * ldb};
#pragma unroll
        for (int im = 0; im < NI; ++im)
#pragma unroll
            for (int q = 0; q < 2; ++q) load_lds(rows + im * apart, bytes, at[q] + col[im], tile + im * TILE + (q * 4 + wave) * 1024);
    }
    __device__ __forceinline__ void fetch_qk(const uint16_t* rows, int64_t ld, int64_t map_stride, int d, int left, XVA_LDS uint8_t* tile, int wave) const {
        fetch(rows, ld, NI == 2 ? map_stride : 0, NI == 2 ? d : map_stride + d, qk, left, tile, wave);
    }
    __device__ __forceinline__ void fetch_v(const uint16_t* rows, int64_t ld, int d, int left, XVA_LDS uint8_t* tile, int wave) const {
        fetch(rows, ld, 0, 2 * d, v, left, tile, wave);
    }
};
// `lane`, but unknown to the compiler: what is computed from it inside a loop is not kept in registers across the loop (where the accumulators leave none)
__device__ __forceinline__ int again(int lane) { asm volatile("" : "+v"(lane)); return lane; }
// LDS offsets of this lane's fragments.  A fragment's other 32-column half and its other 16-column tiles are an XOR away (the swizzle XORs windows, attn_tile.h).
struct Lane {
    uint32_t kc, tr;
    __device__ __forceinline__ Lane(int lane, uint32_t at) { Frag fr; fr.init(lane); kc = fr.kc[0] + at; tr = fr.tr[0] + at; }
    // as Frag's, of image `im` of a buffer: rows it * 16 .. + 15 / columns dt * 16 .. + 15 of rows 32 t ..
    __device__ __forceinline__ bf16x8 rows(const XVA_LDS uint8_t* smem, int im, int it, int kh) const {
        return *reinterpret_cast<const XVA_LDS bf16x8*>(smem + (kc ^ (kh * 64)) + (im * TILE + it * 2048));
    }
    __device__ __forceinline__ bf16x8 cols(const XVA_LDS uint8_t* smem, int im, int dt, int t) const {
        const XVA_LDS uint8_t* a = smem + (tr ^ (dt * 32)) + (im * TILE + t * 4096);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((XVA_LDS s16x4*)a), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((XVA_LDS s16x4*)(a + 2048));
        return __builtin_bit_cast(bf16x8, (s16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};
// 8 elements at column d0 of a row as an MFMA operand, zero behind `width`
__device__ __forceinline__ bf16x8 ld_edge(const uint16_t* row, int d0, int width) {
    const uint4 z = {0, 0, 0, 0};
    return __builtin_bit_cast(bf16x8, d0 < width ? *reinterpret_cast<const uint4*>(row + d0) : z);
}
// image and 32-column half of MFMA step kh of map m
template <int NI> __device__ __forceinline__ int qk_image(int m) { return NI == 2 ? m : 0; }
template <int NI> __device__ __forceinline__ int qk_half(int m, int kh) { return NI == 2 ? kh : m; }
// image and 16-column tile of d tile dt of map m
template <int NI> __device__ __forceinline__ int qk_tile(int m, int dt) { return NI == 2 ? dt : m * 2 + dt; }

// Tiles 0 .. n - 1 with their two LDS buffers by turns.  The buffers are two arrays and the loop is written out for both, so that the compiler sees that the
// reads of one tile do not touch the bytes that the next tile's loads are bringing in, and does not wait for those before the reads.
#define XVA_TWO_BUFFERS(n, tile)                                                          \
    for (int two = 0; two < (n); two += 2) {                                              \
        tile(two, (const XVA_LDS uint8_t*)even, (XVA_LDS uint8_t*)odd);                   \
        if (two + 1 < (n)) tile(two + 1, (const XVA_LDS uint8_t*)odd, (XVA_LDS uint8_t*)even); \
    }
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
#define MFMA(x, y, z) mma16<F16>(x, y, z)
#define ZERO4 ((f32x4){0.f, 0.f, 0.f, 0.f})
// p[i] of an input that is the same in every lane, by a scalar load (a vector load would be waited for together with the tiles in flight)
__device__ __forceinline__ float uniform(const float* p, int i) { return reinterpret_cast<const __attribute__((address_space(4))) float*>((uintptr_t)p)[i]; }
__device__ __forceinline__ float lam_of(const Args& a, int h) {
    return a.lam_type == 0 ? static_cast<const float*>(a.lam)[h] : (a.lam_type == 1 ? ld16<false>(a.lam, h) : ld16<true>(a.lam, h));
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Workgroups that walk over more than this start by their length: ranking the items takes a microsecond or two (32 x 150, heads of 32: 16 -> 22 us of dK / dV / dq)
constexpr int LONG = 512;
// The r-th longest item of a ragged batch, by `lens` (the same in every lane): workgroups start in this order, so that the last ones to start are short (32 x 860 ragged
// frames, 4 heads of 48: forward 90 -> 81 us, dK / dV / dq 183 -> 156).  Each lane ranks one item; larger batches, whose workgroups are many, keep their order.
__device__ __forceinline__ int item_by_length(const int32_t* lens, int B, int T, int r) {
    if (!lens || B > 64 || T <= LONG) return r;
    const int lane = threadIdx.x & 63, mine = lane < B ? len_of(lens, lane, T) : -1;
    int rank = 0;
    for (int j = 0; j < B; ++j) {
        const int other = __builtin_amdgcn_readlane(mine, j);
        rank += other > mine || (other == mine && j < lane);
    }
    return __builtin_ctzll(__ballot(lane < B && rank == r));
}
// A workgroup's block of a (item, head) and its piece.  All pairs over LT long rows: the items by length, with all their blocks; otherwise block by block, under `causal` by
// their length (`last_first`: the last ones see most keys), the items by length within.
struct Block {
    int b, h, blk, piece, blocks;
    __device__ __forceinline__ Block(const Args& a, unsigned id, int heads, int T, int size, const int32_t* lens, int LT, bool last_first) {
        const bool by_block = a.causal || LT <= LONG;
        blocks = (T + size - 1) / size;
        const unsigned all = (unsigned)blocks * a.B * heads;
        piece = id / all;
        const unsigned at = id - piece * all, inner = by_block ? (unsigned)a.B * heads : (unsigned)blocks * heads;
        const int outer = at / inner, in = at - outer * inner, mid = in / heads;
        h = in - mid * heads;
        blk = by_block ? outer : mid;
        b = item_by_length(lens, a.B, LT, by_block ? mid : outer);
        if (last_first) blk = blocks - 1 - blk;
    }
};
// 64-key tiles that some query of the block from q0 on sees
__device__ __forceinline__ int key_tiles(const Args& a, int q0, int ql, int kl, int size = 128) {
    if (q0 >= ql) return 0;
    return ((a.causal ? max(min(kl, min(q0 + size - 1, ql - 1) + kl - ql + 1), 0) : kl) + 63) / 64;
}

// ================================================================================ forward ====
// Running maxima are of c S (base 2).  Before a row's first key: so low that any score moves it, and finite, so that differences need no special case.
constexpr float UNSEEN = -3e38f;
// the largest of eight scores: the IEEE maximum, since fmaxf would first quiet each matrix product's result, an instruction apiece
__device__ __forceinline__ float top8(f32x4 a, f32x4 b) {
#define MAXIMUM __builtin_elementwise_maximum
    return MAXIMUM(MAXIMUM(MAXIMUM(MAXIMUM(a[0], a[1]), a[2]), MAXIMUM(MAXIMUM(a[3], b[0]), b[1])), MAXIMUM(b[2], b[3]));
#undef MAXIMUM
}
// HALF: 64 queries to a workgroup, two waves to 32 of them, each with the first or the second 32 keys of a tile; their softmaxes join through LDS.  For heads of 24 and
// 32, where its 145 registers let a third wave onto each SIMD (forward kernel, us, 128 | 64 queries: 12 items of 860, 4 heads of 32 45 | 38, causal 35 | 27; 16 heads, 8192
// 622 | 583; of 48: 32 items 108 | 116; of 16: 64 items of 1000 147 | 167, 8 heads, 2 x 8192 causal 277 | 258).
__host__ __device__ constexpr int forward_rows(int d16) { return d16 == 2 ? 64 : 128; }       // queries of a workgroup
template <int D16, bool F16, bool TRAIN>
__global__ __launch_bounds__(256, 2) void fwd_kernel(Args a) {
    using S = Shape<D16>;
    constexpr int NI = S::NI;
    __shared__ __attribute__((aligned(1024))) uint8_t even[2 * NI * TILE], odd[2 * NI * TILE];       // {K V} of the even and of the odd tiles (see XVA_TWO_BUFFERS)
    constexpr int SIZE = forward_rows(D16);
    constexpr bool HALF = SIZE == 64;
    constexpr int STEPS = HALF ? 1 : 2;                                       // 32-key steps of a wave in a tile
    const Block qb(a, blockIdx.x, a.H, a.Tq, SIZE, a.kl, a.Tk, true);
    const int h = qb.h, b = qb.b, q0 = qb.blk * SIZE;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, i = lane & 15;
    const int ql = len_of(a.ql, b, a.Tq), kl = len_of(a.kl, b, a.Tk), off = kl - ql, hk = h / a.share;
    const uint16_t* kp = a.k + b * a.kb + hk * a.kh;
    const uint16_t* vp = a.v + b * a.vb + hk * a.vh;
    const uint16_t* qp = a.q + b * a.qb + h * a.qh;
    const int wrow = q0 + (HALF ? wave & 1 : wave) * 32, t0 = HALF ? wave >> 1 : 0;
    // keys that some query of the wave sees, and that every query of the wave sees
    auto seen_by = [&](int row) { return a.causal ? max(min(kl, row + off + 1), 0) : kl; };
    const int wave_keys = wrow < ql ? seen_by(min(wrow + 31, ql - 1)) : 0;
    const int whole_keys = seen_by(wrow);
    const int all = key_tiles(a, q0, ql, kl, SIZE), first = qb.piece * a.qpiece, tiles = min(all - first, a.qpiece);
    if (qb.piece > 0 && tiles <= 0) return;
    Lane fr(lane, t0 * 4096);
    bf16x8 qf[2][2][S::KH];
    // keys that row tile rt's row of this lane sees
    auto limit = [&](int rt) { const int row = wrow + rt * 16 + (again(lane) & 15); return row < ql ? seen_by(row) : 0; };
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
        const int row = wrow + rt * 16 + i;
        const uint16_t* qr = qp + (int64_t)min(row, max(ql - 1, 0)) * a.qt;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int kh = 0; kh < S::KH; ++kh) qf[m][rt][kh] = tiles > 0 ? ld_edge(qr + m * a.qm, kh * 32 + g * 8, a.d) : ld_edge(qr, 1, 0);
    }
    f32x4 o[2][2][S::VT];
    float mx[2][2], sum[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
            mx[m][rt] = UNSEEN; sum[m][rt] = 0.f;
#pragma unroll
            for (int dt = 0; dt < S::VT; ++dt) o[m][rt][dt] = ZERO4;
        }
    if (tiles > 0) {
        const Src<NI> src(lane, wave, a.d, a.km);
        const int row0 = first * 64;
        src.fetch_qk(kp + row0 * a.kt, a.kt, a.km, a.d, kl - row0, (XVA_LDS uint8_t*)even, wave);
        src.fetch_v(vp + row0 * a.vt, a.vt, a.d, kl - row0, (XVA_LDS uint8_t*)even + NI * TILE, wave);
    }
    __syncthreads();
    auto tile = [&](const int it, const XVA_LDS uint8_t* smem, XVA_LDS uint8_t* next) {
        const int jb = first + it;
        if (it + 1 < tiles) {
            const Src<NI> src(again(lane), wave, a.d, a.km);
            const int row0 = (jb + 1) * 64;
            src.fetch_qk(kp + row0 * a.kt, a.kt, a.km, a.d, kl - row0, next, wave);
            src.fetch_v(vp + row0 * a.vt, a.vt, a.d, kl - row0, next + NI * TILE, wave);
        }
        if (jb * 64 + t0 * 32 < wave_keys) {
            const bool whole = (jb + 1) * 64 <= whole_keys;
#pragma unroll
            for (int t = 0; t < STEPS; ++t) {                 // 32 keys at a time
                bf16x8 pf[2][2];
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    f32x4 s[2][2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        s[0][u] = ZERO4; s[1][u] = ZERO4;
#pragma unroll
                        for (int kh = 0; kh < S::KH; ++kh) {
                            const bf16x8 kf = fr.rows(smem, qk_image<NI>(m), 2 * t + u, qk_half<NI>(m, kh));
                            s[0][u] = MFMA(kf, qf[m][0][kh], s[0][u]);         // [key g * 4 + r][row lane & 15]
                            s[1][u] = MFMA(kf, qf[m][1][kh], s[1][u]);
                        }
                    }
                    if (!whole) {
#pragma unroll
                        for (int rt = 0; rt < 2; ++rt) {
                            const int left = limit(rt) - (jb * 64 + (t0 + t) * 32 + g * 4);
#pragma unroll
                            for (int u = 0; u < 2; ++u)
#pragma unroll
                                for (int r = 0; r < 4; ++r) s[rt][u][r] = u * 16 + r < left ? s[rt][u][r] : -INFINITY;
                        }
                    }
                    float top[2];                             // of this lane's keys
#pragma unroll
                    for (int rt = 0; rt < 2; ++rt) top[rt] = top8(s[rt][0], s[rt][1]);
                    if (__any(__builtin_fmaf(top[0], a.c, -mx[m][0]) > 8.f || __builtin_fmaf(top[1], a.c, -mx[m][1]) > 8.f)) {
#pragma unroll
                        for (int rt = 0; rt < 2; ++rt) {
                            float now = fmaxf(top[rt], __shfl_xor(top[rt], 16, 64));
                            now = fmaxf(fmaxf(now, __shfl_xor(now, 32, 64)) * a.c, mx[m][rt]);
                            const float alpha = exp2_(mx[m][rt] - now);
                            mx[m][rt] = now;
                            sum[m][rt] *= alpha;
#pragma unroll
                            for (int dt = 0; dt < S::VT; ++dt) o[m][rt][dt] *= alpha;
                        }
                    }
#pragma unroll
                    for (int rt = 0; rt < 2; ++rt) {
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float p = exp2_(__builtin_fmaf(s[rt][u][r], a.c, -mx[m][rt]));
                                sum[m][rt] += p;
                                s[rt][u][r] = p;
                            }
                        pf[m][rt] = pack_rows<F16>(s[rt][0], s[rt][1]);
                    }
                }
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int dt = 0; dt < S::VT; ++dt) {
                    const bf16x8 vf = fr.cols(smem, NI + (dt >> 2), dt & 3, t);
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int rt = 0; rt < 2; ++rt) o[m][rt][dt] = MFMA(vf, pf[m][rt], o[m][rt][dt]);        // [column g * 4 + r][row lane & 15]
                }
                __builtin_amdgcn_s_setprio(0);
            }
        }
        __syncthreads();
    };
    XVA_TWO_BUFFERS(tiles, tile)
    if constexpr (HALF) {                                     // (the tile loop has ended with a barrier)
        XVA_LDS float* x = (XVA_LDS float*)((wave & 1) ? odd : even) + again(lane);       // [map][max, sum, 4 VT sums] of each lane, a row tile at a time
        constexpr int EACH = 2 + 4 * S::VT;
        static_assert(2 * EACH * 256 <= (int)sizeof even, "half of a wave's state in one buffer");
#pragma unroll
        for (int rt = 0; rt < 2; ++rt) {
            if (wave >> 1) {
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    x[m * EACH * 64] = mx[m][rt]; x[(m * EACH + 1) * 64] = sum[m][rt];
#pragma unroll
                    for (int e = 0; e < 4 * S::VT; ++e) x[(m * EACH + 2 + e) * 64] = o[m][rt][e >> 2][e & 3];
                }
            }
            __syncthreads();
            if (!(wave >> 1)) {
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const float other = x[m * EACH * 64], now = fmaxf(mx[m][rt], other), mine = exp2_(mx[m][rt] - now), its = exp2_(other - now);
                    mx[m][rt] = now;
                    sum[m][rt] = sum[m][rt] * mine + x[(m * EACH + 1) * 64] * its;
#pragma unroll
                    for (int e = 0; e < 4 * S::VT; ++e) o[m][rt][e >> 2][e & 3] = o[m][rt][e >> 2][e & 3] * mine + x[(m * EACH + 2 + e) * 64] * its;
                }
            }
            __syncthreads();
        }
        if (wave >> 1) return;
    }
    const float lam = lam_of(a, h);
    const int w = 2 * a.d;
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
        const int row = wrow + rt * 16 + i;
        const bool seen = limit(rt) > 0;
        float inv[2], total[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            float l = sum[m][rt];
            l += __shfl_xor(l, 16, 64);
            l += __shfl_xor(l, 32, 64);
            total[m] = l;
            inv[m] = seen ? 1.f / l : 0.f;
            if (TRAIN && all <= a.qpiece && g == 0 && row < a.Tq) a.lse[(((int64_t)m * a.B + b) * a.H + h) * a.Tq + row] = seen ? -(mx[m][rt] + __log2f(l)) / a.c : -INFINITY;
        }
        if (all > a.qpiece) {                                  // a piece: (max, sum) of both maps and the sums as they are, for fwd_join_kernel
            if (row >= a.Tq) continue;
            float* to = a.qpart + ((((int64_t)qb.piece * a.B + b) * a.Tq + row) * a.H + h) * (2 * w + 4);
            if (g == 0) *reinterpret_cast<f32x4*>(to) = (f32x4){mx[0][rt], total[0], mx[1][rt], total[1]};
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int dt = 0; dt < S::VT; ++dt)
                    if (dt * 16 + g * 4 < w) *reinterpret_cast<f32x4*>(to + 4 + m * w + dt * 16 + g * 4) = o[m][rt][dt];
            continue;
        }
        if (row >= a.Tq) continue;
        uint16_t* out = a.out + b * a.ob + row * a.ot + h * a.oh;
        uint16_t* m0 = TRAIN ? a.maps + (((int64_t)b * a.Tq + row) * a.H + h) * w : nullptr;
        const int64_t plane = (int64_t)a.B * a.Tq * a.H * w;
#pragma unroll
        for (int dt = 0; dt < S::VT; ++dt) {
            const int col = dt * 16 + g * 4;
            if (col >= w) continue;
            float u[4], v[4], r[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                u[e] = seen ? o[0][rt][dt][e] * inv[0] : 0.f;
                v[e] = seen ? o[1][rt][dt][e] * inv[1] : 0.f;
                r[e] = u[e] - lam * v[e];
            }
            *reinterpret_cast<uint2*>(out + col) = make_uint2(pack2<F16>(r[0], r[1]), pack2<F16>(r[2], r[3]));
            if (TRAIN) {
                *reinterpret_cast<uint2*>(m0 + col) = make_uint2(pack2<F16>(u[0], u[1]), pack2<F16>(u[2], u[3]));
                *reinterpret_cast<uint2*>(m0 + plane + col) = make_uint2(pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3]));
            }
        }
    }
}

// joins the pieces of a row: four columns to a thread
template <bool F16>
__global__ __launch_bounds__(256) void fwd_join_kernel(Args a) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)a.B * a.Tq * a.H;
    const int w = 2 * a.d, quads = w / 4;
    const int64_t R = id / quads;
    if (R >= rows) return;
    const int col = (int)(id - R * quads) * 4, h = (int)(R % a.H), b = (int)(R / ((int64_t)a.Tq * a.H)), row = (int)(R / a.H - (int64_t)b * a.Tq);
    const int ql = len_of(a.ql, b, a.Tq), kl = len_of(a.kl, b, a.Tk), size = forward_rows((a.d + 15) / 16), all = key_tiles(a, row & -size, ql, kl, size);
    if (all <= a.qpiece) return;
    const float* from = a.qpart + R * (2 * w + 4);
    const int64_t step = rows * (2 * w + 4);
    const int n = (all + a.qpiece - 1) / a.qpiece;
    float mx[2] = {UNSEEN, UNSEEN}, sum[2] = {0.f, 0.f};
    f32x4 o[2] = {ZERO4, ZERO4};
#pragma unroll 4
    for (int p = 0; p < n; ++p)
#pragma unroll
        for (int m = 0; m < 2; ++m) mx[m] = fmaxf(mx[m], from[p * step + 2 * m]);
#pragma unroll 4
    for (int p = 0; p < n; ++p) {
        const f32x4 st = *reinterpret_cast<const f32x4*>(from + p * step);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const float by = exp2_(st[2 * m] - mx[m]);         // (a piece of which nothing is seen: its sums are zero, or no numbers where its scores are none)
            sum[m] += st[2 * m + 1] * by;
            o[m] += *reinterpret_cast<const f32x4*>(from + p * step + 4 + m * w + col) * by;
        }
    }
    const bool seen = row < ql && (!a.causal || row + kl - ql >= 0);
    const float lam = lam_of(a, h);
    const f32x4 u = seen ? o[0] * (1.f / sum[0]) : ZERO4, v = seen ? o[1] * (1.f / sum[1]) : ZERO4;
    xva_attn::st4<F16>(a.out + b * a.ob + row * a.ot + h * a.oh + col, seen ? u - v * lam : ZERO4, 1.f);
    if (a.maps) {
        xva_attn::st4<F16>(a.maps + R * w + col, u, 1.f);
        xva_attn::st4<F16>(a.maps + (rows + R) * w + col, v, 1.f);
        if (col < 8) {
            const int m = col >> 2;
            a.lse[(((int64_t)m * a.B + b) * a.H + h) * a.Tq + row] = seen ? -(mx[m] + __log2f(sum[m])) / a.c : -INFINITY;
        }
    }
}

// ================================================================================ forward, few queries ====
// Up to 32 rows (query heads of a key head x queries) against a long cache: the work is reading k and v once, so the rows of all heads that share a key head sit
// in one matrix tile and the keys are what is cut up.  A workgroup takes a chunk of keys, its waves the chunk's 32-key tiles by turns, each with its own softmax
// and its own buffers (nothing waits for another wave): k straight to registers in the fragments' layout, v through LDS for its transposed fragments, both one
// tile ahead.  The waves' results join in LDS, the chunks' (where there are several) in a second kernel.
// Partial results of a chunk: (max, sum) of [2][rows], then [2][rows][2 d] sums of exp2(c (S - max)) V.
template <int D16, bool F16, int RT>
__global__ __launch_bounds__(256, RT == 2 && D16 >= 3 ? 1 : 2) void few_kernel(Args a, float* __restrict__ part, int chunk, int nsplit) {
    using S = Shape<D16>;
    constexpr int NI = S::NI, HALF = TILE / 2, W = NI * 64;                    // bytes of a 32-row image; padded width of v
    __shared__ __attribute__((aligned(1024))) uint8_t even[4 * NI * HALF], odd[4 * NI * HALF];
    __shared__ float stat[4][2][RT * 16][2];
    const int split = blockIdx.x % nsplit, bh = blockIdx.x / nsplit, hk = bh % a.Hk, b = bh / a.Hk;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, i = lane & 15, w = 2 * a.d, R = a.share * a.Tq;
    const int ql = len_of(a.ql, b, a.Tq), kl = len_of(a.kl, b, a.Tk), off = kl - ql;
    const int k0 = split * chunk, k1 = min(k0 + chunk, kl);
    const uint16_t* kp = a.k + b * a.kb + hk * a.kh;
    const uint16_t* vp = a.v + b * a.vb + hk * a.vh;
    bf16x8 qf[2][RT][S::KH];
    int limit[RT];                                                             // keys that the lane's row sees
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = rt * 16 + i, hs = r / a.Tq, t = r - hs * a.Tq;
        const bool row = r < R && t < ql;
        limit[rt] = row ? (a.causal ? max(min(kl, t + off + 1), 0) : kl) : 0;
        const uint16_t* qr = a.q + b * a.qb + (row ? t : 0) * a.qt + (hk * a.share + (row ? hs : 0)) * a.qh;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int kh = 0; kh < S::KH; ++kh) qf[m][rt][kh] = ld_edge(qr + m * a.qm, kh * 32 + g * 8, row ? a.d : 0);
    }
    f32x4 o[2][RT][S::VT];
    float mx[2][RT], sum[2][RT];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            mx[m][rt] = -INFINITY; sum[m][rt] = 0.f;
#pragma unroll
            for (int dt = 0; dt < S::VT; ++dt) o[m][rt][dt] = ZERO4;
        }
    const Lane fr(lane, wave * NI * HALF);
    bf16x8 kf[2][2][S::KH], kn[2][2][S::KH];                                   // this tile's and the next one's
    auto fetch = [&](int key0, XVA_LDS uint8_t* to, bf16x8 (&into)[2][2][S::KH]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint16_t* row = kp + (int64_t)min(key0 + u * 16 + i, k1 - 1) * a.kt;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int kh = 0; kh < S::KH; ++kh) {
                    const int d0 = kh * 32 + g * 8;                            // (behind d: columns that meet q's zeros; a load on every way, see below)
                    into[m][u][kh] = xva_attn::ld_frag(row + m * a.km + (d0 < a.d ? d0 : 0));
                }
        }
        const int p = lane & 7;
        const uint32_t left = max(k1 - key0, 1), ldb = (uint32_t)a.vt * 2u, bytes = (min(left, 32u) - 1) * ldb + w * 2;
        const uint16_t* rows = vp + min(key0, k1 - 1) * a.vt;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t r = q * 8 + (lane >> 3), c = (((p >> 1) ^ ((r >> 1) & 3)) << 1) | (p & 1);
#pragma unroll
            for (int im = 0; im < NI; ++im) {
                const int e0 = im * 64 + c * 8;
                load_lds(rows, bytes, min(r, left - 1) * ldb + 2 * (e0 < w ? e0 : 0), to + (wave * NI + im) * HALF + q * 1024);
            }
        }
    };
    auto tile = [&](int key0, const XVA_LDS uint8_t* smem, XVA_LDS uint8_t* next, bf16x8 (&kc)[2][2][S::KH], bf16x8 (&kx)[2][2][S::KH]) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                     // the other buffer's last reads have arrived
        fetch(key0 + 128, next, kx);
        bf16x8 pf[2][RT];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            f32x4 s[RT][2];
            bool grew = false;
            float top[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    s[rt][u] = ZERO4;
#pragma unroll
                    for (int kh = 0; kh < S::KH; ++kh) s[rt][u] = MFMA(kc[m][u][kh], qf[m][rt][kh], s[rt][u]);       // [key g * 4 + r][row lane & 15]
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[rt][u][r] = key0 + u * 16 + g * 4 + r < min(limit[rt], k1) ? s[rt][u][r] : -INFINITY;
                }
                top[rt] = fmaxf(fmaxf(fmaxf(s[rt][0][0], s[rt][0][1]), fmaxf(s[rt][0][2], s[rt][0][3])),
                                fmaxf(fmaxf(s[rt][1][0], s[rt][1][1]), fmaxf(s[rt][1][2], s[rt][1][3])));
                grew |= (top[rt] - mx[m][rt]) * a.c > 8.f;
            }
            if (__any(grew)) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    float now = fmaxf(top[rt], __shfl_xor(top[rt], 16, 64));
                    now = fmaxf(fmaxf(now, __shfl_xor(now, 32, 64)), mx[m][rt]);
                    const float alpha = mx[m][rt] == now ? 1.f : exp2_((mx[m][rt] - now) * a.c);
                    mx[m][rt] = now;
                    sum[m][rt] *= alpha;
#pragma unroll
                    for (int dt = 0; dt < S::VT; ++dt) o[m][rt][dt] *= alpha;
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const float base = mx[m][rt] == -INFINITY ? 0.f : mx[m][rt] * a.c;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float p = exp2_(s[rt][u][r] * a.c - base);
                        sum[m][rt] += p;
                        s[rt][u][r] = p;
                    }
                pf[m][rt] = pack_rows<F16>(s[rt][0], s[rt][1]);
            }
        }
#pragma unroll
        for (int dt = 0; dt < S::VT; ++dt) {
            const XVA_LDS uint8_t* at = smem + (fr.tr ^ ((dt & 3) * 32)) + (dt >> 2) * HALF;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((XVA_LDS s16x4*)at), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((XVA_LDS s16x4*)(at + 2048));
            const bf16x8 vf = __builtin_bit_cast(bf16x8, (s16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) o[m][rt][dt] = MFMA(vf, pf[m][rt], o[m][rt][dt]);                    // [column g * 4 + r][row lane & 15]
        }
    };
    const int mine = k0 + wave * 32;
    // A tile is fetched behind the last one too (its rows clamped to the chunk's last): on every way through the loop the same number of loads is in flight, so
    // that the compiler can wait for the older ones alone.
    if (mine < k1) {
        fetch(mine, (XVA_LDS uint8_t*)even, kf);
        for (int key0 = mine;; key0 += 256) {
            tile(key0, (const XVA_LDS uint8_t*)even, (XVA_LDS uint8_t*)odd, kf, kn);
            if (key0 + 128 >= k1) break;
            tile(key0 + 128, (const XVA_LDS uint8_t*)odd, (XVA_LDS uint8_t*)even, kn, kf);
            if (key0 + 256 >= k1) break;
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                           // (the last fetch's bytes land before the buffers are used for the results)
    // the waves' maxima and sums
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float l = sum[m][rt];
            l += __shfl_xor(l, 16, 64);
            l += __shfl_xor(l, 32, 64);
            if (g == 0) { stat[wave][m][rt * 16 + i][0] = mx[m][rt]; stat[wave][m][rt * 16 + i][1] = l; }
        }
    __syncthreads();
    // a map and 16 rows at a time: every wave's sums relative to the common maximum, [wave][row][column] in LDS, added and taken on by 16 x 16 threads
    XVA_LDS float* x = (XVA_LDS float*)even;
    const int row = threadIdx.x >> 4, col = (threadIdx.x & 15) * (W / 16);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float first[W / 16];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            float top = -INFINITY;
#pragma unroll
            for (int v = 0; v < 4; ++v) top = fmaxf(top, stat[v][m][rt * 16 + i][0]);
            const float scale = mx[m][rt] == -INFINITY ? 0.f : exp2_((mx[m][rt] - top) * a.c);
#pragma unroll
            for (int dt = 0; dt < S::VT; ++dt) *reinterpret_cast<XVA_LDS f32x4*>(x + (wave * 16 + i) * W + dt * 16 + g * 4) = o[m][rt][dt] * scale;
            __syncthreads();
            const int r = rt * 16 + row;
            float rtop = -INFINITY, l = 0.f, acc[W / 16];
#pragma unroll
            for (int v = 0; v < 4; ++v) rtop = fmaxf(rtop, stat[v][m][r][0]);
#pragma unroll
            for (int v = 0; v < 4; ++v) l += stat[v][m][r][1] * (stat[v][m][r][0] == -INFINITY ? 0.f : exp2_((stat[v][m][r][0] - rtop) * a.c));
#pragma unroll
            for (int e = 0; e < W / 16; ++e) acc[e] = x[row * W + col + e] + x[(16 + row) * W + col + e] + x[(32 + row) * W + col + e] + x[(48 + row) * W + col + e];
            if (r < R && col < w) {
                if (nsplit > 1) {
                    float* to = part + (int64_t)blockIdx.x * 2 * R * (w + 2);
                    if (col == 0) { to[(m * R + r) * 2] = rtop; to[(m * R + r) * 2 + 1] = l; }
#pragma unroll
                    for (int e = 0; e < W / 16; ++e)
                        if (col + e < w) to[4 * R + (int64_t)(m * R + r) * w + col + e] = acc[e];
                } else {
                    const float inv = l == 0.f ? 0.f : 1.f / l;                // (nothing seen; scores that are no numbers have a sum, which is none)
                    if (m == 0) {
#pragma unroll
                        for (int e = 0; e < W / 16; ++e) first[e] = acc[e] * inv;
                    } else {
                        const int hs = r / a.Tq, h = hk * a.share + hs;
                        const float by = lam_of(a, h);
                        uint16_t* out = a.out + b * a.ob + (int64_t)(r - hs * a.Tq) * a.ot + h * a.oh;
#pragma unroll
                        for (int e = 0; e < W / 16; e += 2)
                            if (col + e < w)
                                *reinterpret_cast<uint32_t*>(out + col + e) = pack2<F16>(first[e] - by * acc[e] * inv,
                                                                                         first[e + 1] - by * acc[e + 1] * inv);
                    }
                }
            }
            __syncthreads();
        }
    }
}

// joins the chunks of a row: weights of the chunks first, into LDS, then eight slots of chunks beside each other over the columns (four to a thread)
constexpr int MAX_SPLIT = 1024;
template <bool F16>
__global__ __launch_bounds__(256) void few_join_kernel(Args a, const float* __restrict__ part, int nsplit) {
    __shared__ float by[2][MAX_SPLIT], sh[16];
    __shared__ f32x4 sums[2][8][32];
    const int w = 2 * a.d, R = a.share * a.Tq;
    const int id = blockIdx.x, bh = id / R, r = id - bh * R, hk = bh % a.Hk, b = bh / a.Hk;
    const int64_t each = (int64_t)2 * R * (w + 2);
    const float* p = part + (int64_t)bh * nsplit * each;
    float inv[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        float top = -INFINITY, l = 0.f;
        for (int k = threadIdx.x; k < nsplit; k += 256) top = fmaxf(top, by[m][k] = p[k * each + (m * R + r) * 2]);
        top = xva_block_max(top, sh);
        for (int k = threadIdx.x; k < nsplit; k += 256) {
            const float e = by[m][k] == -INFINITY ? 0.f : exp2_((by[m][k] - top) * a.c);
            by[m][k] = e;
            l += e * p[k * each + (m * R + r) * 2 + 1];
        }
        l = xva_block_sum(l, sh);
        inv[m] = top == -INFINITY ? 0.f : 1.f / l;
    }
    __syncthreads();
    const int slot = threadIdx.x >> 5, col = (threadIdx.x & 31) * 4;
    if (col < w) {
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            f32x4 acc = ZERO4;
            const float* q = p + 4 * R + (int64_t)(m * R + r) * w + col;
#pragma unroll 4
            for (int k = slot; k < nsplit; k += 8)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] += q[k * each + e] * by[m][k];
            sums[m][slot][threadIdx.x & 31] = acc;
        }
    }
    __syncthreads();
    if (slot == 0 && col < w) {
        f32x4 t[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            t[m] = sums[m][0][threadIdx.x];
#pragma unroll
            for (int k = 1; k < 8; ++k) t[m] += sums[m][k][threadIdx.x];
            t[m] *= inv[m];
        }
        const int hs = r / a.Tq, h = hk * a.share + hs;
        xva_attn::st4<F16>(a.out + b * a.ob + (int64_t)(r - hs * a.Tq) * a.ot + h * a.oh + col, t[0] - lam_of(a, h) * t[1], 1.f);
    }
}

// ================================================================================ backward ====
// D_m[row] = dO . O_m; 16 lanes to a row of 2 d <= 128 columns.  fp16: a workgroup's rows are 16 of one head, and it leaves the largest squared norm of dO among them; the
// workgroups from `first_v` on leave that of 16 of v's rows.
template <bool F16>
__global__ __launch_bounds__(256) void rowdot_kernel(Args a, unsigned first_v) {
    __shared__ float top[4];
    const int slot = threadIdx.x >> 4, c = (threadIdx.x & 15) * 8, w = 2 * a.d;
    const bool keys = F16 && blockIdx.x >= first_v;
    int64_t id;                                    // of the row in (B, Tq, H)
    int b, h, t;
    bool row;
    if constexpr (F16) {
        const int T = keys ? a.Tk : a.Tq, heads = keys ? a.Hk : a.H, blocks = (T + 15) / 16;
        const unsigned at = blockIdx.x - (keys ? first_v : 0), bh = at / (unsigned)blocks;
        b = bh / (unsigned)heads; h = bh - b * heads; t = (at - bh * blocks) * 16 + slot;
        row = t < T;
        id = ((int64_t)b * T + t) * heads + h;
    } else {
        id = (int64_t)blockIdx.x * 16 + slot;
        row = id < (int64_t)a.B * a.Tq * a.H;
        const int64_t bt = id / a.H;
        h = (int)(id - bt * a.H); b = (int)(bt / a.Tq); t = (int)(bt - (int64_t)b * a.Tq);
    }
    const int64_t rows = (int64_t)a.B * a.Tq * a.H;
    float s[2] = {0.f, 0.f}, n = 0.f;
    if (row && c < w && t < (keys ? len_of(a.kl, b, a.Tk) : len_of(a.ql, b, a.Tq))) {
        const uint4 gr = *reinterpret_cast<const uint4*>((keys ? a.v + b * a.vb + t * a.vt + h * a.vh : a.dout + b * a.gb + t * a.gt + h * a.gh) + c);
        const uint32_t gw[4] = {gr.x, gr.y, gr.z, gr.w};
        if (F16) {
#pragma unroll
            for (int e = 0; e < 4; ++e) { float g0, g1; unpack2<F16>(gw[e], g0, g1); n += g0 * g0 + g1 * g1; }
        }
        if (!keys) {
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const uint4 od = *reinterpret_cast<const uint4*>(a.maps + (m * rows + id) * w + c);
                const uint32_t ow[4] = {od.x, od.y, od.z, od.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float g0, g1, o0, o1;
                    unpack2<F16>(gw[e], g0, g1); unpack2<F16>(ow[e], o0, o1);
                    s[m] += g0 * o0 + g1 * o1;
                }
            }
        }
    }
    auto join = [](float v) { v += __shfl_xor(v, 1, 64); v += __shfl_xor(v, 2, 64); v += __shfl_xor(v, 4, 64); return v + __shfl_xor(v, 8, 64); };
    if (!keys) {
#pragma unroll
        for (int m = 0; m < 2; ++m) s[m] = join(s[m]);
        if (row && (threadIdx.x & 15) < 2) a.D[(((int64_t)(threadIdx.x & 1) * a.B + b) * a.H + h) * a.Tq + t] = threadIdx.x & 1 ? s[0] - s[1] : -s[0];
        const int64_t first = (int64_t)blockIdx.x * 16 + slot;
        if (first < a.H && (threadIdx.x & 15) == 0) a.lam32[first] = lam_of(a, (int)first);
    }
    if constexpr (F16) {
        n = join(n);
        n = fmaxf(n, __shfl_xor(n, 16, 64));
        n = fmaxf(n, __shfl_xor(n, 32, 64));
        if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = n;
        __syncthreads();
        if (threadIdx.x == 0) a.norms[blockIdx.x] = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    }
}

// fp16 holds 2^-14 .. 2^16 in full: dS = P (dP - D) of a loss that is a mean over many values, or lam times it, lies below that and would be lost, and one of large
// gradients above it.  |dS| <= |dP - D| <= 2 max |dO_i| max |v_j| (norms over the 2 d columns), so 2^U brings it to at most 2^15; 2^el >= |lam|.  All factors are powers of
// two, undone in fp32 where sums are rounded.  One set for all that adds up in a key head's dK, so an item whose gradients are small beside another's keeps its own.
//   dq : dS 2^U in the sum that takes D off (no product more).
//   dkv: U > 0 in the exponents, P 2^kp, as far as P_1 - lam P_2 has room, 14 - el powers; U < 0 in v and D (2^kv).  Both are in the rows' logsumexp and D that it starts its
//        products from (`start`), so its loop has no product more; dS_2 takes lam / 2^el instead of lam.  (A product for each pair instead: 4 - 5 % of the kernel;
//        kp beside the exponent's factor: two constants where an instruction takes one from the scalar unit, registers spill.)
// (860 keys, heads of 48, dO of 1e-3, lam 0.01: dk_2 off by 9 % of its norm without this.  It costs 8 us of 224, forward
// and backward, on 32 x 860 frames: v's norms and a launch.)  A gradient or value that is not finite takes no factor: the results it reaches
// are lost as they are.
struct Range {
    float up, down;                               // 2^U, 2^-U
    float el, big, shrink;                        // el, 2^el, 2^kv
    float undo_k, undo_v, unused;                 // 2^-(kp + kv), 2^-kp
    template <bool F16> static __device__ __forceinline__ Range of(const Args& a, int b, int hk) {
        if constexpr (!F16) return {1.f, 1.f, 0.f, 1.f, 1.f, 1.f, 1.f, 0.f};
        else {
            const int at = (b * a.Hk + hk) * 8;
            auto e = [&](int i) { return uniform(a.range, at + i); };
            return {e(0), e(1), e(2), e(3), e(4), e(5), e(6), 0.f};
        }
    }
};
// The range of an (item, key head), which every workgroup finds for itself from the few norms there are, and what dkv's products start from: (4, B, H, Tq), the
// logsumexps of both maps, then D, with the range's factors.  A workgroup: 256 rows of a head, under way while it looks for the norms' maxima.
__global__ __launch_bounds__(256) void range_kernel(Args a) {
    __shared__ float top[3][4];
    const int parts = (a.Tq + 255) / 256, bh = blockIdx.x / parts, part = blockIdx.x - bh * parts, b = bh / a.H, h = bh - b * a.H, hk = h / a.share;
    const int64_t rows = (int64_t)a.B * a.H * a.Tq, at = (int64_t)bh * a.Tq + part * 256 + threadIdx.x;
    const bool row = part * 256 + (int)threadIdx.x < a.Tq;
    float from[4];
#pragma unroll
    for (int m = 0; m < 2; ++m) { from[m] = row ? a.lse[m * rows + at] : 0.f; from[2 + m] = row ? a.D[m * rows + at] : 0.f; }
    const int nq = (a.Tq + 15) / 16, nk = (a.Tk + 15) / 16;
    const float* g = a.norms + ((int64_t)b * a.H + hk * a.share) * nq;
    const float* v = a.norms + (int64_t)a.B * a.H * nq + ((int64_t)b * a.Hk + hk) * nk;
    float mg = 0.f, mv = 0.f, lam = 0.f;
    for (int e = threadIdx.x; e < a.share * nq; e += 256) mg = fmaxf(mg, g[e]);
    for (int e = threadIdx.x; e < nk; e += 256) mv = fmaxf(mv, v[e]);
    for (int e = threadIdx.x; e < a.share; e += 256) lam = fmaxf(lam, fabsf(lam_of(a, hk * a.share + e)));
    mg = xva_wave_max(mg); mv = xva_wave_max(mv); lam = xva_wave_max(lam);
    if ((threadIdx.x & 63) == 0) { const int w = threadIdx.x >> 6; top[0][w] = mg; top[1][w] = mv; top[2][w] = lam; }
    __syncthreads();
    auto all = [&](int i) { return fmaxf(fmaxf(top[i][0], top[i][1]), fmaxf(top[i][2], top[i][3])); };
    mg = all(0); mv = all(1); lam = all(2);
    const float bound = 2.002f * sqrtf(mg) * sqrtf(mv);             // (2 and some roundings)
    int up = 0, el = 0;
    if (bound > 0.f && bound < INFINITY) { frexpf(bound, &up); up = 15 - up; }
    if (lam > 0.f && lam < INFINITY) { frexpf(lam, &el); el = max(el, -100); }
    const int kp = min(max(up, 0), 14 - max(el, 0)), kv = min(up, 0);
    if (threadIdx.x == 0 && part == 0 && h == hk * a.share)
        *reinterpret_cast<Range*>(a.range + ((int64_t)b * a.Hk + hk) * 8) = {ldexpf(1.f, up), ldexpf(1.f, -up), (float)el, ldexpf(1.f, el), ldexpf(1.f, kv), ldexpf(1.f, -kp - kv),
                                                                            ldexpf(1.f, -kp), 0.f};
    const float more = (float)kp / a.c, shrink = ldexpf(1.f, kv);
    if (!row) return;
#pragma unroll
    for (int m = 0; m < 2; ++m) { a.start[m * rows + at] = from[m] + more; a.start[(2 + m) * rows + at] = from[2 + m] * shrink; }
}

// A key block's 64-query tiles: of each query head that shares the keys, `per_head` from tile `t0` on
struct KeyBlock {
    int t0, per_head, all;
    __device__ __forceinline__ KeyBlock(const Args& a, int k0, int ql, int kl) {
        const int first = a.causal ? max(k0 - (kl - ql), 0) : 0;       // queries that see a key of the block: from here on
        t0 = first / 64;
        per_head = k0 < kl && first < ql ? (ql + 63) / 64 - t0 : 0;
        all = per_head * a.share;
    }
};

// dK, dV of 64 keys of a key head over the query heads that share it and their 64-query tiles.  Waves: two halves of the keys x two halves of a tile's
// queries; the queries' halves are added at the end through LDS.  (128 keys to a workgroup, 32 to a wave over all rows: half as many workgroups, which
// leaves long causal sequences waiting for the first keys' ones.)
// Where key blocks are few, or causal ones of very different length, the tiles of a key block are cut into pieces, one to a workgroup; a second kernel adds the pieces'
// fp32 sums in order (rows of [2][d] of dK and [2 d] of dV).  Query blocks' keys are cut the same way in the forward pass and in dq.
template <int D16> struct BwdLds {
    // (the widest heads' accumulators leave too few registers for all of V's fragments: a spilled one would be waited for together with the tiles in flight)
    static constexpr int AWAY = D16 == 4 ? 3 : 0;                                             // V fragments of the second key tile kept in LDS
    static constexpr int STAT = 2 * Shape<D16>::NI * TILE;                                     // {Q dO | lse1 lse2 D1 D2} of the even and of the odd tiles
    typedef uint8_t Buffer[STAT + 1024];
    typedef uint8_t Away[AWAY ? AWAY * 4096 : 16];
};
template <int D16, bool F16>
__device__ __forceinline__ void dkv_part(const Args& a, const unsigned id, typename BwdLds<D16>::Buffer& even, typename BwdLds<D16>::Buffer& odd, typename BwdLds<D16>::Away& away_raw) {
    using S = Shape<D16>;
    constexpr int NI = S::NI, AWAY = BwdLds<D16>::AWAY, STAT = BwdLds<D16>::STAT;
    const Block at(a, id, a.Hk, a.Tk, 64, a.ql, a.Tq, false);             // (under `causal` the first keys are seen by most queries: they start first)
    const int kblk = at.blk, piece = at.piece, hk = at.h, b = at.b, k0 = kblk * 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, i = lane & 15, t = wave >> 1;
    const int ql = len_of(a.ql, b, a.Tq), kl = len_of(a.kl, b, a.Tk), off = kl - ql;
    const int wkey = k0 + (wave & 1) * 32, w = 2 * a.d;
    Lane fr(lane, t * 4096);
    const KeyBlock kb(a, k0, ql, kl);
    const bool any = kb.all > 0;
    const int begin = piece * a.piece, total = min(kb.all - begin, a.piece);
    if (piece > 0 && total <= 0) return;
    const Range range = Range::of<F16>(a, b, hk);
    bf16x8 kf[2][2][S::KH], vf[2][S::VH];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
        const int key = min(wkey + kt * 16 + i, max(kl - 1, 0));
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int kh = 0; kh < S::KH; ++kh) kf[m][kt][kh] = ld_edge(a.k + b * a.kb + hk * a.kh + m * a.km + key * a.kt, kh * 32 + g * 8, any ? a.d : 0);
#pragma unroll
        for (int kh = 0; kh < S::VH; ++kh) vf[kt][kh] = ld_edge(a.v + b * a.vb + hk * a.vh + key * a.vt, kh * 32 + g * 8, any ? w : 0);
    }
    if (F16 && range.shrink != 1.f) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int kh = 0; kh < S::VH; ++kh) {
                u32x4 e = __builtin_bit_cast(u32x4, vf[kt][kh]);
#pragma unroll
                for (int i = 0; i < 4; ++i) { float v0, v1; unpack2<F16>(e[i], v0, v1); e[i] = pack2<F16>(v0 * range.shrink, v1 * range.shrink); }
                vf[kt][kh] = __builtin_bit_cast(bf16x8, e);
            }
    }
    XVA_LDS bf16x8* away = (XVA_LDS bf16x8*)away_raw + wave * AWAY * 64 + lane;
#pragma unroll
    for (int e = 0; e < AWAY; ++e) away[e * 64] = vf[1][S::VH - 1 - e];
    auto v_of = [&](int kt, int kh) { return kt == 1 && kh >= S::VH - AWAY ? away[(S::VH - 1 - kh) * 64] : vf[kt][kh]; };
    f32x4 dk[2][2][S::DT], dv[2][S::VT];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int dt = 0; dt < S::DT; ++dt) dk[m][kt][dt] = ZERO4;
#pragma unroll
        for (int dt = 0; dt < S::VT; ++dt) dv[kt][dt] = ZERO4;
    }
    auto fetch = [&](int hs, int row0, XVA_LDS uint8_t* to) {
        const int h = hk * a.share + hs, lane_ = again(lane);
        const Src<NI> src(lane_, wave, a.d, a.qm);
        src.fetch_qk(a.q + b * a.qb + h * a.qh + row0 * a.qt, a.qt, a.qm, a.d, ql - row0, to, wave);
        src.fetch_v(a.dout + b * a.gb + h * a.gh + row0 * a.gt, a.gt, a.d, ql - row0, to + NI * TILE, wave);
        const float* from = (F16 ? a.start + (int64_t)(wave & 2) * a.B * a.H * a.Tq : wave < 2 ? a.lse : a.D) + (((int64_t)(wave & 1) * a.B + b) * a.H + h) * a.Tq + row0;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void*)from, 0, (uint32_t)min(ql - row0, 64) * 4u, 0x00027000),
                                                 (XVA_LDS void*)(to + STAT + wave * 256), 4, min(lane_, ql - row0 - 1) * 4, 0, 0, 0);
    };
    // from the last rows on, which all key blocks see, and by turns over the heads: workgroups that start together read the same tiles at about the same time
    int qtile = kb.t0 + kb.per_head - 1 - begin / a.share, hs = begin % a.share;
    if (any) fetch(hs, qtile * 64, (XVA_LDS uint8_t*)even);
    __syncthreads();
    auto tile = [&](const int it, const XVA_LDS uint8_t* smem, XVA_LDS uint8_t* next) {
        const int row0 = qtile * 64;
        const float lam = uniform(a.lam32, hk * a.share + hs), loglam = __log2f(fabsf(lam)) - range.el, minus = lam < 0.f ? 1.f : -1.f, minus_big = minus * range.big;
        if (++hs == a.share) { hs = 0; --qtile; }
        if (it + 1 < total) fetch(hs, qtile * 64, next);
        const int wrow = row0 + t * 32;                       // this wave's 32 rows
        const bool whole = wrow + 32 <= ql && wkey + 32 <= kl && (!a.causal || wkey + 31 <= wrow + off);      // every row sees every key
        const bool none = wkey >= kl || wrow >= ql || (a.causal && wkey > wrow + 31 + off);
        if (!none) {
            u32x4 pk[3][2];                                   // P_1 - lam P_2, dS_1, dS_2 of each key tile, 32 rows in the permuted order
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                // -D_1 under dP, lse under the scores
                const XVA_LDS uint8_t* at = smem + STAT + t * 128 + (F16 && D16 == 4 ? again(lane) >> 4 : g) * 16 + u * 64;      // (kept, it would be spilled there)
                const f32x4 nD = *reinterpret_cast<const XVA_LDS f32x4*>(at + 512);
                f32x4 s[2][2], dp[2];                         // [map][key tile], [row g * 4 + r][key lane & 15]
#pragma unroll
                for (int kh = 0; kh < S::VH; ++kh) {
                    const bf16x8 of = fr.rows(smem, NI + (kh >> 1), u, kh & 1);
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt) dp[kt] = MFMA(of, v_of(kt, kh), kh ? dp[kt] : nD);
                }
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const f32x4 nL = *reinterpret_cast<const XVA_LDS f32x4*>(at + m * 256);
#pragma unroll
                    for (int kh = 0; kh < S::KH; ++kh) {
                        const bf16x8 qf = fr.rows(smem, qk_image<NI>(m), u, qk_half<NI>(m, kh));
#pragma unroll
                        for (int kt = 0; kt < 2; ++kt) s[m][kt] = MFMA(qf, kf[m][kt][kh], kh ? s[m][kt] : nL);
                    }
                }
                if (!whole) {
                    const int l = again(lane);
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int row = wrow + u * 16 + (l >> 4) * 4 + r, key = wkey + kt * 16 + (l & 15);
                            const bool ok = (row < ql) & (key < kl) & (!a.causal | (key <= row + off));
                            s[0][kt][r] = ok ? s[0][kt][r] : -INFINITY;
                            s[1][kt][r] = ok ? s[1][kt][r] : -INFINITY;
                        }
                }
                const f32x4 dD = *reinterpret_cast<const XVA_LDS f32x4*>(at + 768) * minus;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        // (|lam| in the exponent, its sign in the sums: no product more than without it)
                        const float p1 = exp2_(s[0][kt][r] * a.c), p2 = exp2_(__builtin_fmaf(s[1][kt][r], a.c, loglam)), x = dp[kt][r];
                        s[0][kt][r] = p1 * x;
                        s[1][kt][r] = p2 * __builtin_fmaf(x, minus, dD[r]);
                        dp[kt][r] = __builtin_fmaf(p2, minus_big, p1);
                    }
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        pk[0][kt][2 * u + e] = pack2<F16>(dp[kt][2 * e], dp[kt][2 * e + 1]);
                        pk[1][kt][2 * u + e] = pack2<F16>(s[0][kt][2 * e], s[0][kt][2 * e + 1]);
                        pk[2][kt][2 * u + e] = pack2<F16>(s[1][kt][2 * e], s[1][kt][2 * e + 1]);
                    }
                __builtin_amdgcn_sched_barrier(0);            // (16 rows at a time: registers)
            }
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int dt = 0; dt < S::VT; ++dt) {
                const bf16x8 of = fr.cols(smem, NI + (dt >> 2), dt & 3, 0);
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) dv[kt][dt] = MFMA(of, __builtin_bit_cast(bf16x8, pk[0][kt]), dv[kt][dt]);                  // [column g * 4 + r][key lane & 15]
            }
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int dt = 0; dt < S::DT; ++dt) {
                    const bf16x8 qf = fr.cols(smem, qk_image<NI>(m), qk_tile<NI>(m, dt), 0);
#pragma unroll
                    for (int kt = 0; kt < 2; ++kt) dk[m][kt][dt] = MFMA(qf, __builtin_bit_cast(bf16x8, pk[1 + m][kt]), dk[m][kt][dt]);
                }
            __builtin_amdgcn_s_setprio(0);
        }
        __syncthreads();
    };
    XVA_TWO_BUFFERS(total, tile)
    const int l = again(lane), ge = l >> 4, ie = l & 15;
    // the second half of the queries hands its sums over: 16 bytes a lane and accumulator
    XVA_LDS f32x4* xch = (XVA_LDS f32x4*)((wave & 1) ? odd : even) + l;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
        if (t == 1) {
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int dt = 0; dt < S::DT; ++dt) xch[(m * S::DT + dt) * 64] = dk[m][kt][dt];
#pragma unroll
            for (int dt = 0; dt < S::VT; ++dt) xch[(2 * S::DT + dt) * 64] = dv[kt][dt];
        }
        __syncthreads();
        const int key = wkey + kt * 16 + ie;
        if (t == 0 && key < a.Tk && kb.all > a.piece) {
            float* row = a.part + (((int64_t)piece * a.B + b) * a.Tk + key) * a.Hk * 4 * a.d + hk * 4 * a.d;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int dt = 0; dt < S::DT; ++dt)
                    if (dt * 16 + ge * 4 < a.d) *reinterpret_cast<f32x4*>(row + m * a.d + dt * 16 + ge * 4) = dk[m][kt][dt] + xch[(m * S::DT + dt) * 64];
#pragma unroll
            for (int dt = 0; dt < S::VT; ++dt)
                if (dt * 16 + ge * 4 < w) *reinterpret_cast<f32x4*>(row + w + dt * 16 + ge * 4) = dv[kt][dt] + xch[(2 * S::DT + dt) * 64];
        } else if (t == 0 && key < a.Tk) {
            const int64_t row = ((int64_t)b * a.Tk + key) * a.Hk + hk;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int dt = 0; dt < S::DT; ++dt)
                    if (dt * 16 + ge * 4 < a.d) xva_attn::st4<F16>(a.dk + (row * 2 + m) * a.d + dt * 16 + ge * 4, dk[m][kt][dt] + xch[(m * S::DT + dt) * 64], a.scale * range.undo_k * (m ? range.big : 1.f));
#pragma unroll
            for (int dt = 0; dt < S::VT; ++dt)
                if (dt * 16 + ge * 4 < w) xva_attn::st4<F16>(a.dv + row * w + dt * 16 + ge * 4, dv[kt][dt] + xch[(2 * S::DT + dt) * 64], range.undo_v);
        }
        __syncthreads();
    }
}

// the pieces of a key's dK and dV, four columns to a thread
template <bool F16>
__global__ __launch_bounds__(256) void dkv_join_kernel(Args a) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)a.B * a.Tk * a.Hk, row = id / a.d;
    if (row >= rows) return;
    const int col = (int)(id - row * a.d) * 4, w = 2 * a.d;
    const int b = (int)(row / ((int64_t)a.Tk * a.Hk)), key = (int)(row / a.Hk - (int64_t)b * a.Tk);
    const KeyBlock kb(a, key & ~63, len_of(a.ql, b, a.Tq), len_of(a.kl, b, a.Tk));
    if (kb.all <= a.piece) return;
    f32x4 v = ZERO4;
    for (int p = 0; p * a.piece < kb.all; ++p) v += *reinterpret_cast<const f32x4*>(a.part + (p * rows + row) * 2 * w + col);
    const float* range = a.range + ((int64_t)b * a.Hk + row % a.Hk) * 8;
    if (col < w) xva_attn::st4<F16>(a.dk + row * w + col, v, F16 ? a.scale * range[5] * (col < a.d ? 1.f : range[3]) : a.scale);
    else xva_attn::st4<F16>(a.dv + row * w + col - w, v, F16 ? range[6] : 1.f);
}

// dq of 128 queries of a head, 32 to a wave, and their part of dlam
template <int D16, bool F16>
__device__ __forceinline__ void dq_part(const Args& a, const unsigned id, typename BwdLds<D16>::Buffer& even, typename BwdLds<D16>::Buffer& odd) {
    using S = Shape<D16>;
    constexpr int NI = S::NI;
    const Block qb(a, id, a.H, a.Tq, 128, a.kl, a.Tk, true);
    const int h = qb.h, b = qb.b, q0 = qb.blk * 128;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, i = lane & 15;
    const int ql = len_of(a.ql, b, a.Tq), kl = len_of(a.kl, b, a.Tk), off = kl - ql, hk = h / a.share;
    const uint16_t* kp = a.k + b * a.kb + hk * a.kh;
    const uint16_t* vp = a.v + b * a.vb + hk * a.vh;
    const int wrow = q0 + wave * 32, w = 2 * a.d;
    auto seen_by = [&](int row) { return a.causal ? max(min(kl, row + off + 1), 0) : kl; };
    const int wave_keys = wrow < ql ? seen_by(min(wrow + 31, ql - 1)) : 0;
    const int whole_keys = seen_by(wrow);
    const int all = key_tiles(a, q0, ql, kl), first = qb.piece * a.qpiece, tiles = min(all - first, a.qpiece);
    if (qb.piece > 0 && tiles <= 0) {
        if (threadIdx.x == 0) a.dlam_part[(((int64_t)h * a.B + b) * qb.blocks + qb.blk) * a.qpieces + qb.piece] = 0.f;
        return;
    }
    Lane fr(lane, 0);
    const Range range = Range::of<F16>(a, b, hk);
    bf16x8 qf[2][2][S::KH], of[2][S::VH];
    int limit[2];
    float L[2][2], Dr[2][2];
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
        const int row = wrow + rt * 16 + i, safe = min(row, max(ql - 1, 0));
        limit[rt] = row < ql ? seen_by(row) : 0;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int kh = 0; kh < S::KH; ++kh) qf[m][rt][kh] = ld_edge(a.q + b * a.qb + h * a.qh + m * a.qm + safe * a.qt, kh * 32 + g * 8, tiles > 0 ? a.d : 0);
            const int64_t at = (((int64_t)m * a.B + b) * a.H + h) * a.Tq + safe;
            L[m][rt] = -a.lse[at] * a.c; Dr[m][rt] = a.D[at];
        }
        Dr[0][rt] = -Dr[0][rt];
        Dr[1][rt] = Dr[0][rt] - Dr[1][rt];
        if (F16) { Dr[0][rt] *= range.up; Dr[1][rt] *= range.up; }
#pragma unroll
        for (int kh = 0; kh < S::VH; ++kh) of[rt][kh] = ld_edge(a.dout + b * a.gb + h * a.gh + safe * a.gt, kh * 32 + g * 8, tiles > 0 ? w : 0);
    }
    f32x4 dq[2][2][S::DT];
    float dl = 0.f;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int rt = 0; rt < 2; ++rt)
#pragma unroll
            for (int dt = 0; dt < S::DT; ++dt) dq[m][rt][dt] = ZERO4;
    if (tiles > 0) {
        const Src<NI> src(lane, wave, a.d, a.km);
        const int row0 = first * 64;
        src.fetch_qk(kp + row0 * a.kt, a.kt, a.km, a.d, kl - row0, (XVA_LDS uint8_t*)even, wave);
        src.fetch_v(vp + row0 * a.vt, a.vt, a.d, kl - row0, (XVA_LDS uint8_t*)even + NI * TILE, wave);
    }
    __syncthreads();
    auto tile = [&](const int it, const XVA_LDS uint8_t* smem, XVA_LDS uint8_t* next) {
        const int jb = first + it;
        if (it + 1 < tiles) {
            const Src<NI> src(again(lane), wave, a.d, a.km);
            const int row0 = (jb + 1) * 64;
            src.fetch_qk(kp + row0 * a.kt, a.kt, a.km, a.d, kl - row0, next, wave);
            src.fetch_v(vp + row0 * a.vt, a.vt, a.d, kl - row0, next + NI * TILE, wave);
        }
        if (jb * 64 < wave_keys) {
            const bool whole = (jb + 1) * 64 <= whole_keys && wrow + 32 <= ql;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f32x4 s[2][2][2], dp[2][2];                 // [map][key tile][row tile], [key g * 4 + r][row lane & 15]
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int kt = 2 * t + u;
#pragma unroll
                    for (int rt = 0; rt < 2; ++rt) { s[0][u][rt] = ZERO4; s[1][u][rt] = ZERO4; dp[u][rt] = ZERO4; }
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int kh = 0; kh < S::KH; ++kh) {
                            const bf16x8 kf = fr.rows(smem, qk_image<NI>(m), kt, qk_half<NI>(m, kh));
#pragma unroll
                            for (int rt = 0; rt < 2; ++rt) s[m][u][rt] = MFMA(kf, qf[m][rt][kh], s[m][u][rt]);
                        }
#pragma unroll
                    for (int kh = 0; kh < S::VH; ++kh) {
                        const bf16x8 vf = fr.rows(smem, NI + (kh >> 1), kt, kh & 1);
#pragma unroll
                        for (int rt = 0; rt < 2; ++rt) dp[u][rt] = MFMA(vf, of[rt][kh], dp[u][rt]);
                    }
                    if (!whole) {
#pragma unroll
                        for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const bool ok = jb * 64 + kt * 16 + g * 4 + r < limit[rt];
                                s[0][u][rt][r] = ok ? s[0][u][rt][r] : -INFINITY;
                                s[1][u][rt][r] = ok ? s[1][u][rt][r] : -INFINITY;
                            }
                    }
#pragma unroll
                    for (int rt = 0; rt < 2; ++rt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float p1 = exp2_(s[0][u][rt][r] * a.c - L[0][rt]), p2 = exp2_(s[1][u][rt][r] * a.c - L[1][rt]);
                            const float x = dp[u][rt][r];
                            dl += p2 * x;
                            s[0][u][rt][r] = p1 * (F16 ? __builtin_fmaf(x, range.up, -Dr[0][rt]) : x - Dr[0][rt]);
                            s[1][u][rt][r] = p2 * (F16 ? __builtin_fmaf(x, range.up, -Dr[1][rt]) : x - Dr[1][rt]);
                        }
                }
                bf16x8 df[2][2];
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int rt = 0; rt < 2; ++rt) df[m][rt] = pack_rows<F16>(s[m][0][rt], s[m][1][rt]);
                __builtin_amdgcn_s_setprio(1);
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int dt = 0; dt < S::DT; ++dt) {
                        const bf16x8 kf = fr.cols(smem, qk_image<NI>(m), qk_tile<NI>(m, dt), t);
#pragma unroll
                        for (int rt = 0; rt < 2; ++rt) dq[m][rt][dt] = MFMA(kf, df[m][rt], dq[m][rt][dt]);       // [column g * 4 + r][row lane & 15]
                    }
                __builtin_amdgcn_s_setprio(0);
            }
        }
        __syncthreads();
    };
    XVA_TWO_BUFFERS(tiles, tile)
    const float lam = uniform(a.lam32, h);
#pragma unroll
    for (int rt = 0; rt < 2; ++rt) {
        const int row = wrow + rt * 16 + i;
        if (row >= a.Tq) continue;
        if (all > a.qpiece) {                                  // a piece, for dq_join_kernel
            float* to = a.qpart + ((((int64_t)qb.piece * a.B + b) * a.Tq + row) * a.H + h) * w;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int dt = 0; dt < S::DT; ++dt)
                    if (dt * 16 + g * 4 < a.d) *reinterpret_cast<f32x4*>(to + m * a.d + dt * 16 + g * 4) = dq[m][rt][dt];
            continue;
        }
        uint16_t* dst = a.dq + (((int64_t)b * a.Tq + row) * a.H + h) * w;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int dt = 0; dt < S::DT; ++dt)
                if (dt * 16 + g * 4 < a.d) xva_attn::st4<F16>(dst + m * a.d + dt * 16 + g * 4, dq[m][rt][dt], (m ? -lam * a.scale : a.scale) * range.down);
    }
    // (the tile loop has ended with a barrier)
    XVA_LDS float* red = (XVA_LDS float*)even;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) dl += __shfl_xor(dl, o, 64);
    if (lane == 0) red[wave] = dl;
    __syncthreads();
    if (threadIdx.x == 0) a.dlam_part[(((int64_t)h * a.B + b) * qb.blocks + qb.blk) * a.qpieces + qb.piece] = red[0] + red[1] + red[2] + red[3];
}

// One launch for both: the first `dkv` workgroups take key blocks, the others query blocks, which fill the chip where the last key blocks leave it empty (32 x 860
// frames, heads of 48: 128 + 84 us in two launches, 178 in one; 8192 causal positions, heads of 64: 1095 | 1073).
template <int D16, bool F16>
__global__ __launch_bounds__(256, 2) void grad_kernel(Args a, unsigned dkv) {
    __shared__ __attribute__((aligned(1024))) typename BwdLds<D16>::Buffer even, odd;
    __shared__ __attribute__((aligned(16))) typename BwdLds<D16>::Away away;
    if (blockIdx.x < dkv) dkv_part<D16, F16>(a, blockIdx.x, even, odd, away);
    else dq_part<D16, F16>(a, blockIdx.x - dkv, even, odd);
}

// the pieces of a row's dq, four columns to a thread
template <bool F16>
__global__ __launch_bounds__(256) void dq_join_kernel(Args a) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, rows = (int64_t)a.B * a.Tq * a.H;
    const int w = 2 * a.d, quads = w / 4;
    const int64_t R = id / quads;
    if (R >= rows) return;
    const int col = (int)(id - R * quads) * 4, h = (int)(R % a.H), b = (int)(R / ((int64_t)a.Tq * a.H)), row = (int)(R / a.H - (int64_t)b * a.Tq);
    const int all = key_tiles(a, row & ~127, len_of(a.ql, b, a.Tq), len_of(a.kl, b, a.Tk));
    if (all <= a.qpiece) return;
    f32x4 v = ZERO4;
    for (int p = 0; p * a.qpiece < all; ++p) v += *reinterpret_cast<const f32x4*>(a.qpart + (p * rows + R) * w + col);
    xva_attn::st4<F16>(a.dq + R * w + col, v, (col < a.d ? a.scale : -a.lam32[h] * a.scale) * (F16 ? a.range[((int64_t)b * a.Hk + h / a.share) * 8 + 1] : 1.f));
}

// dlam[h] = - sum of the head's parts, in a fixed order, rounded once to lam's type
__global__ __launch_bounds__(256) void dlam_kernel(const float* __restrict__ part, void* __restrict__ dlam, int type, int n) {
    __shared__ float sh[16];
    float v = 0.f;
    for (int k = threadIdx.x; k < n; k += 256) v += part[(int64_t)blockIdx.x * n + k];
    v = xva_block_sum(v, sh);
    if (threadIdx.x != 0) return;
    if (type == 0) static_cast<float*>(dlam)[blockIdx.x] = -v;
    else static_cast<uint16_t*>(dlam)[blockIdx.x] = type == 1 ? cvt16<false>(-v) : cvt16<true>(-v);
}
#undef MFMA

// -------------------------------------------------------------------------------- host ----
int check(const xva_diff_attention_args* p, const char* who) {
    XVA_CHECK_ARG(p, "%s: null argument", who);
    XVA_CHECK_ARG(p->dtype == 1 || p->dtype == 2, "%s: dtype %d (bf16 or fp16)", who, p->dtype);
    XVA_CHECK_ARG(p->B >= 0 && p->Tq >= 0 && p->Tk >= 0 && p->Tq < (1 << 30) && p->Tk < (1 << 30) && p->H >= 1 && p->Hk >= 1 && p->H % p->Hk == 0,
                  "%s: B %d Tq %d Tk %d H %d Hk %d", who, p->B, p->Tq, p->Tk, p->H, p->Hk);
    XVA_CHECK_ARG(p->d >= 8 && p->d <= 64 && p->d % 8 == 0, "%s: head width %d (a multiple of 8 up to 64)", who, p->d);
    XVA_CHECK_ARG(p->scale > 0.f, "%s: scale %g", who, p->scale);
    XVA_CHECK_ARG(p->lam_dtype >= 0 && p->lam_dtype <= 2, "%s: lam of dtype %d", who, p->lam_dtype);
    if (p->B == 0 || p->Tq == 0) return XVA_OK;
    XVA_CHECK_ARG(p->q && p->lam && (p->Tk == 0 || (p->k && p->v)), "%s: null argument", who);
    uintptr_t ptrs = (uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->out | (uintptr_t)p->dout;
    int64_t all = 0;
    for (int e = 0; e < 4; ++e) all |= p->q_stride[e] | p->k_stride[e];
    for (int e = 0; e < 3; ++e) all |= p->v_stride[e] | p->out_stride[e] | p->dout_stride[e];
    // 64 rows of a tile, and its maps, within 32-bit byte offsets
    const int64_t near[] = {p->q_stride[1], p->q_stride[3], p->k_stride[1], p->k_stride[3], p->v_stride[1], p->dout_stride[1]};
    for (int64_t e : near) XVA_CHECK_ARG(e >= 0 && e < (1 << 24), "%s: row and map strides are 0 .. 2^24 - 1", who);
    XVA_CHECK_ARG(ptrs % 16 == 0 && all % 8 == 0, "%s: addresses are 16-byte aligned and strides multiples of 8", who);
    const int64_t wgs = (int64_t)p->B * p->H * ((p->Tq + 63) / 64), kwgs = (int64_t)p->B * p->Hk * ((p->Tk + 63) / 64);
    XVA_CHECK_ARG(xva_seq::launchable(wgs + kwgs, 256), "%s: too many blocks", who);
    return XVA_OK;
}
Args args_of(const xva_diff_attention_args* p) {
    Args a = {};
    a.q = (const uint16_t*)p->q; a.k = (const uint16_t*)p->k; a.v = (const uint16_t*)p->v; a.dout = (const uint16_t*)p->dout;
    a.out = (uint16_t*)p->out; a.maps = (uint16_t*)p->maps; a.dq = (uint16_t*)p->dq; a.dk = (uint16_t*)p->dk; a.dv = (uint16_t*)p->dv;
    a.lam = p->lam; a.lam_type = p->lam_dtype; a.lse = p->lse; a.ql = p->q_lens; a.kl = p->k_lens;
    a.qb = p->q_stride[0]; a.qt = p->q_stride[1]; a.qh = p->q_stride[2]; a.qm = p->q_stride[3];
    a.kb = p->k_stride[0]; a.kt = p->k_stride[1]; a.kh = p->k_stride[2]; a.km = p->k_stride[3];
    a.vb = p->v_stride[0]; a.vt = p->v_stride[1]; a.vh = p->v_stride[2];
    a.ob = p->out_stride[0]; a.ot = p->out_stride[1]; a.oh = p->out_stride[2];
    a.gb = p->dout_stride[0]; a.gt = p->dout_stride[1]; a.gh = p->dout_stride[2];
    a.B = p->B; a.Tq = p->Tq; a.Tk = p->Tk; a.H = p->H; a.Hk = p->Hk; a.share = p->H / p->Hk; a.d = p->d; a.causal = p->causal;
    a.scale = p->scale; a.c = p->scale * 1.44269504088896341f;
    return a;
}
// Few rows: keys of a chunk, a multiple of the 128 that the four waves take in one turn; about 1024 workgroups (four to a CU: items of a ragged batch end early),
// none with less than 128 keys
struct Few { bool on; int chunk, nsplit; };
Few few_plan(const xva_diff_attention_args* p) {
    Few f = {p->maps == nullptr && (int64_t)p->H / p->Hk * p->Tq <= 32 && p->Tk > 0 && p->B > 0 && p->Tq > 0, 0, 1};
    if (!f.on) return f;
    const int64_t heads = (int64_t)p->B * p->Hk, want = (1024 + heads - 1) / heads;
    int64_t chunk = (p->Tk + want - 1) / want;
    chunk = (chunk + 127) / 128 * 128;
    f.chunk = (int)chunk;
    f.nsplit = (int)((p->Tk + chunk - 1) / chunk);
    return f;
}
int64_t few_floats(const xva_diff_attention_args* p, const Few& f) {
    return f.on && f.nsplit > 1 ? (int64_t)p->B * p->H * p->Tq * f.nsplit * 2 * (2 * p->d + 2) : 0;
}
template <int D16, bool F16> int few(const Args& a, const Few& f, float* part, hipStream_t st) {
    const unsigned grid = (unsigned)(a.B * a.Hk * f.nsplit);
    if (a.share * a.Tq <= 16) few_kernel<D16, F16, 1><<<grid, 256, 0, st>>>(a, part, f.chunk, f.nsplit);
    else few_kernel<D16, F16, 2><<<grid, 256, 0, st>>>(a, part, f.chunk, f.nsplit);
    XVA_LAUNCH_CHECK();
    if (f.nsplit > 1) {
        few_join_kernel<F16><<<(unsigned)(a.B * a.H * a.Tq), 256, 0, st>>>(a, part, f.nsplit);
        XVA_LAUNCH_CHECK();
    }
    return XVA_OK;
}
// Pieces of the tiles that a workgroup would walk over: 512 workgroups are on the card at once, and `wgs` are fewer than that, or `causal` makes their lengths (up to
// `most` tiles) differ.  All pairs: as many pieces as fill the card.  `causal`: pieces of one length, 512 in all.  Four tiles long at least; a piece's sums are written
// and read once more, so the cut pays where workgroups are at most `few`, or `causal` ones long and less than `uneven`.
// Uncut | cut, us, with the joining kernel:
//   dkv, heads of 64: 16 heads on 4 keys', 8192 positions, causal (512 workgroups) 865 | 701 (pieces of half that length 767); 4 heads, 4096, all pairs (256) 125 | 99
//   (half that length 110); 5 items of 2635 on 391, one head (35) 90 | 27
//   forward + dq: one item of 860, 4 heads of 64 (28) 77 | 46; 10 items of 232 on 3397, 3 heads of 48 (60) 228 | 85; 6 items of 860, 4 heads of 32 (168) 64 | 62; 8 of
//   them (224) 65 | 72; 8 heads of 64, 4096, causal (256) 286 | 227; 12 items of 860, 4 heads of 32, causal (336, of 14 tiles) 66 | 76
struct Pieces { int pieces, piece; };
Pieces pieces_of(int64_t wgs, int64_t most, bool causal, int few, int uneven) {
    Pieces s = {1, (int)(most < 1 ? 1 : most)};
    if (wgs == 0 || wgs > (causal && most >= 32 ? uneven : few)) return s;
    int64_t piece = causal ? (most * wgs + 1023) / 1024 : (most + 512 / wgs - 1) / (512 / wgs);
    if (piece < 4) piece = 4;
    if (piece < most) { s.piece = (int)piece; s.pieces = (int)((most + piece - 1) / piece); }
    return s;
}
Pieces dkv_plan(const xva_diff_attention_args* p) {
    return pieces_of((int64_t)p->B * p->Hk * ((p->Tk + 63) / 64), (int64_t)(p->H / p->Hk) * ((p->Tq + 63) / 64), p->causal, 256, 768);
}
Pieces query_plan(const xva_diff_attention_args* p, bool bwd) {
    const int rows = bwd ? 128 : forward_rows((p->d + 15) / 16);
    return pieces_of((int64_t)p->B * p->H * ((p->Tq + rows - 1) / rows), (p->Tk + 63) / 64, p->causal, 192, 512);
}
int64_t dkv_floats(const xva_diff_attention_args* p) {
    const Pieces s = dkv_plan(p);
    return s.pieces > 1 ? (int64_t)s.pieces * p->B * p->Tk * p->Hk * 4 * p->d : 0;
}
int64_t query_floats(const xva_diff_attention_args* p, bool bwd) {
    const Pieces s = query_plan(p, bwd);
    return s.pieces > 1 ? (int64_t)s.pieces * p->B * p->Tq * p->H * (bwd ? 2 * p->d : 4 * p->d + 4) : 0;
}
int64_t norm_floats(const xva_diff_attention_args* p) { return p->dtype == 2 ? (int64_t)p->B * p->H * ((p->Tq + 15) / 16) + (int64_t)p->B * p->Hk * ((p->Tk + 15) / 16) : 0; }
int64_t range_floats(const xva_diff_attention_args* p) { return p->dtype == 2 ? (int64_t)p->B * p->Hk * 8 : 0; }
int64_t start_floats(const xva_diff_attention_args* p) { return p->dtype == 2 ? (int64_t)4 * p->B * p->H * p->Tq : 0; }
unsigned join_grid(const Args& a) { return (unsigned)(((int64_t)a.B * a.Tq * a.H * (a.d / 2) + 255) / 256); }
template <int D16, bool F16> int forward(const Args& a, bool train, hipStream_t st) {
    const unsigned grid = (unsigned)(a.B * a.H * ((a.Tq + forward_rows(D16) - 1) / forward_rows(D16)) * a.qpieces);
    if (train) fwd_kernel<D16, F16, true><<<grid, 256, 0, st>>>(a);
    else fwd_kernel<D16, F16, false><<<grid, 256, 0, st>>>(a);
    XVA_LAUNCH_CHECK();
    if (a.qpieces > 1) {
        fwd_join_kernel<F16><<<join_grid(a), 256, 0, st>>>(a);
        XVA_LAUNCH_CHECK();
    }
    return XVA_OK;
}
template <int D16, bool F16> int backward(const Args& a, void* dlam, hipStream_t st) {
    const int nqb = (a.Tq + 127) / 128;
    const int64_t rows = (int64_t)a.B * a.Tq * a.H;
    const unsigned first_v = F16 ? (unsigned)((int64_t)a.B * a.H * ((a.Tq + 15) / 16)) : (unsigned)((rows + 15) / 16);
    rowdot_kernel<F16><<<first_v + (F16 ? (unsigned)((int64_t)a.B * a.Hk * ((a.Tk + 15) / 16)) : 0), 256, 0, st>>>(a, first_v);
    XVA_LAUNCH_CHECK();
    if (F16) {
        range_kernel<<<(unsigned)((int64_t)a.B * a.H * ((a.Tq + 255) / 256)), 256, 0, st>>>(a);
        XVA_LAUNCH_CHECK();
    }
    const unsigned dkv = (unsigned)(a.B * a.Hk * ((a.Tk + 63) / 64) * a.pieces);
    grad_kernel<D16, F16><<<dkv + (unsigned)(a.B * a.H * nqb * a.qpieces), 256, 0, st>>>(a, dkv);
    XVA_LAUNCH_CHECK();
    if (a.pieces > 1) {
        dkv_join_kernel<F16><<<(unsigned)(((int64_t)a.B * a.Tk * a.Hk * a.d + 255) / 256), 256, 0, st>>>(a);
        XVA_LAUNCH_CHECK();
    }
    if (a.qpieces > 1) {
        dq_join_kernel<F16><<<join_grid(a), 256, 0, st>>>(a);
        XVA_LAUNCH_CHECK();
    }
    dlam_kernel<<<a.H, 256, 0, st>>>(a.dlam_part, dlam, a.lam_type, a.B * nqb * a.qpieces);
    XVA_LAUNCH_CHECK();
    return XVA_OK;
}
int64_t workspace(const xva_diff_attention_args* p, bool bwd) {
    const Few f = few_plan(p);
    if (!bwd) return (f.on ? few_floats(p, f) : query_floats(p, false)) * 4;
    return (dkv_floats(p) + query_floats(p, true) + range_floats(p) + start_floats(p) + norm_floats(p) + (int64_t)2 * p->B * p->H * p->Tq + (int64_t)p->H * p->B * ((p->Tq + 127) / 128) * query_plan(p, true).pieces + p->H) * 4;
}
}   // namespace

extern "C" int64_t xva_diff_attention_workspace_bytes(const xva_diff_attention_args* p, int backward_pass) {
    return p && p->B >= 0 && p->Tq >= 0 && p->Tk >= 0 && p->H >= 1 && p->Hk >= 1 && p->H % p->Hk == 0 ? workspace(p, backward_pass != 0) : -1;
}

#define XVA_DIFF_BY_SHAPE(call)                                                          \
    switch ((p->d + 15) / 16 * 2 + (p->dtype == 2)) {                                    \
        case 2: return call(1, false); case 3: return call(1, true);                     \
        case 4: return call(2, false); case 5: return call(2, true);                     \
        case 6: return call(3, false); case 7: return call(3, true);                     \
        case 8: return call(4, false); default: return call(4, true);                    \
    }

extern "C" int xva_diff_attention_fwd(const xva_diff_attention_args* p, void* ws, int64_t ws_bytes, void* stream) {
    XVA_TRY(check(p, "xva_diff_attention_fwd"));
    if (p->B == 0 || p->Tq == 0) return XVA_OK;
    XVA_CHECK_ARG(p->out && (p->maps == nullptr) == (p->lse == nullptr), "xva_diff_attention_fwd: null argument");
    Args a = args_of(p);
    const Few f = few_plan(p);
    XVA_CHECK_ARG(xva_seq::launchable((int64_t)p->B * p->Hk * f.nsplit, 256) && (f.nsplit == 1 || xva_seq::launchable((int64_t)p->B * p->H * p->Tq, 256)),
                  "xva_diff_attention_fwd: too many blocks");
    const Pieces s = query_plan(p, false);
    a.qpieces = s.pieces; a.qpiece = s.piece; a.qpart = (float*)ws;
    const int64_t need = workspace(p, false);
    if (ws_bytes < need || (need && !ws)) {
        xva_set_error("xva_diff_attention_fwd: workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)need);
        return XVA_ERR_WS;
    }
#define CALL(D16, F16) (f.on ? few<D16, F16>(a, f, (float*)ws, (hipStream_t)stream) : forward<D16, F16>(a, p->maps != nullptr, (hipStream_t)stream))
    XVA_DIFF_BY_SHAPE(CALL)
#undef CALL
}
extern "C" int xva_diff_attention_bwd(const xva_diff_attention_args* p, void* ws, int64_t ws_bytes, void* stream) {
    XVA_TRY(check(p, "xva_diff_attention_bwd"));
    if (p->B == 0 || p->Tq == 0) return XVA_OK;
    XVA_CHECK_ARG(p->dout && p->maps && p->lse && p->dq && p->dlam && (p->Tk == 0 || (p->dk && p->dv)), "xva_diff_attention_bwd: null argument");
    XVA_CHECK_ARG(xva_seq::launchable((int64_t)p->B * p->H * ((p->Tq + 15) / 16) + (int64_t)p->B * p->Hk * ((p->Tk + 15) / 16), 256),
                  "xva_diff_attention_bwd: too many rows");
    if (ws_bytes < workspace(p, true) || !ws) {
        xva_set_error("xva_diff_attention_bwd: workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)workspace(p, true));
        return XVA_ERR_WS;
    }
    Args a = args_of(p);
    const Pieces s = dkv_plan(p);
    const Pieces sq = query_plan(p, true);
    a.pieces = s.pieces; a.piece = s.piece; a.qpieces = sq.pieces; a.qpiece = sq.piece;
    a.part = (float*)ws;
    a.qpart = a.part + dkv_floats(p);
    a.range = a.qpart + query_floats(p, true);
    a.start = a.range + range_floats(p);
    a.norms = a.start + start_floats(p);
    a.D = a.norms + norm_floats(p);
    a.dlam_part = a.D + (int64_t)2 * p->B * p->H * p->Tq;
    a.lam32 = a.dlam_part + (int64_t)p->H * p->B * ((p->Tq + 127) / 128) * a.qpieces;
#define CALL(D16, F16) backward<D16, F16>(a, p->dlam, (hipStream_t)stream)
    XVA_DIFF_BY_SHAPE(CALL)
#undef CALL
}
