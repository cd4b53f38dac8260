// attn_tile.h — the [64 rows][64 columns] 16-bit LDS tile of the attention kernels and its MFMA fragments (gfx950).
//
// The LDS image XORs the 32-byte window of a row with (row >> 1) & 3, which makes BOTH access patterns conflict-free: ds_read_b128 MFMA fragments along the
// columns (Q K^T, dO V^T) and ds_read_b64_tr_b16 transposed fragments along the rows (P V, dS^T Q, P^T dO, dS K).
// MFMA convention: mfma(X, Y) with X = fragment indexed a, Y = fragment indexed b gives every lane the outputs [a = (lane >> 4) * 4 + r][b = lane & 15].
#pragma once
#include "gemm_glds.h"

namespace xva_attn {
using namespace xva_glds;

constexpr int TILE = 64 * 64 * 2;   // bytes of one LDS tile

__device__ __forceinline__ uint32_t chunk_off(int r, int c) { return r * 128 + (((((c >> 1) ^ ((r >> 1) & 3)) << 1) | (c & 1)) << 4); }

struct Frag {
    uint32_t kc[2];   // ds_read_b128 fragment (index = row tile, k = head dim): lane offset for kh = 0, 1
    uint32_t tr[4];   // transpose-read fragment (index = column tile dt, k = rows): lane offset for dt = 0..3
    __device__ __forceinline__ void init(int lane) {
        const int g = lane >> 4, i = lane & 15;
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) kc[kh] = chunk_off(i, kh * 4 + g);
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) tr[dt] = chunk_off(g * 4 + (i >> 2), dt * 2 + ((i & 3) >> 1)) + (i & 1) * 8;
    }
    // rows it*16 .. +15 of the tile as an MFMA operand indexed by row, k = kh*32 + (lane>>4)*8 + e
    __device__ __forceinline__ bf16x8 read_kc(const XVA_LDS uint8_t* tile, int it, int kh) const {
        return *reinterpret_cast<const XVA_LDS bf16x8*>(tile + it * 2048 + kc[kh]);
    }
    // columns dt*16 .. +15 as an MFMA operand indexed by column; k-step t covers rows 32t .. 32t+31 in the PERMUTED order
    // e < 4: row 32t + (lane>>4)*4 + e ; e >= 4: row 32t + 16 + (lane>>4)*4 + (e-4)   (matches pack_rows below)
    __device__ __forceinline__ bf16x8 read_tr(const XVA_LDS uint8_t* tile, int dt, int t) const {
        const XVA_LDS uint8_t* a = tile + t * 4096 + tr[dt];
        s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((XVA_LDS s16x4*)a);
        s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((XVA_LDS s16x4*)(a + 2048));
        return __builtin_bit_cast(bf16x8, (s16x8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
};

// two accumulator tiles (rows / keys 32t + g*4 + r and 32t + 16 + g*4 + r) -> one bf16 operand in the permuted k order
// (F16: the 16-bit format of every tensor and MFMA operand of the kernel — false bf16, true IEEE half; gemm_glds.h)
template <bool F16 = false>
__device__ __forceinline__ bf16x8 pack_rows(f32x4 a, f32x4 b) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    u32x4 v = {pack2<F16>(a[0], a[1]), pack2<F16>(a[2], a[3]), pack2<F16>(b[0], b[1]), pack2<F16>(b[2], b[3])};
    return __builtin_bit_cast(bf16x8, v);
}
__device__ __forceinline__ bf16x8 ld_frag(const uint16_t* p) { return __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(p)); }
template <bool F16 = false>
__device__ __forceinline__ void st4(uint16_t* dst, f32x4 v, float s) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<F16>(v[0] * s, v[1] * s), pack2<F16>(v[2] * s, v[3] * s));
}
}   // namespace xva_attn
