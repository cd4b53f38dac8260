// seq_vec.h — vector loads and stores of a sequence tensor's element types (0 fp32, 1 bf16, 2 fp16) as fp32 registers.
#pragma once
#include "gemm_glds.h"

namespace xva_seq {
using xva_glds::cvt16;
using xva_glds::pack2;
using xva_glds::unpack2;

// V elements of the 16-bit or fp32 type DT (0 fp32, 1 bf16, 2 fp16) <-> registers
template <int DT, int V> __device__ __forceinline__ void load_v(const void* base, int64_t off, float (&f)[V]) {
    if constexpr (DT == 0) {
        const float* p = reinterpret_cast<const float*>(base) + off;
        if constexpr (V >= 4) {
#pragma unroll
            for (int e = 0; e < V; e += 4) { const float4 v = *reinterpret_cast<const float4*>(p + e); f[e] = v.x; f[e + 1] = v.y; f[e + 2] = v.z; f[e + 3] = v.w; }
        } else if constexpr (V == 2) { const float2 v = *reinterpret_cast<const float2*>(p); f[0] = v.x; f[1] = v.y; }
        else f[0] = p[0];
    } else {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(base) + off;
        if constexpr (V == 1) f[0] = xva_glds::ld16<DT == 2>(base, off);
        else {
            uint32_t w[V / 2];
            if constexpr (V >= 8) {
#pragma unroll
                for (int e = 0; e < V / 8; ++e) { const uint4 v = reinterpret_cast<const uint4*>(p)[e]; w[4 * e] = v.x; w[4 * e + 1] = v.y; w[4 * e + 2] = v.z; w[4 * e + 3] = v.w; }
            } else if constexpr (V == 4) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
            else w[0] = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
            for (int e = 0; e < V / 2; ++e) unpack2<DT == 2>(w[e], f[2 * e], f[2 * e + 1]);
        }
    }
}
template <int DT, int V> __device__ __forceinline__ void store_v(void* base, int64_t off, const float (&f)[V]) {
    if constexpr (DT == 0) {
        float* p = reinterpret_cast<float*>(base) + off;
        if constexpr (V >= 4) {
#pragma unroll
            for (int e = 0; e < V; e += 4) *reinterpret_cast<float4*>(p + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
        } else if constexpr (V == 2) *reinterpret_cast<float2*>(p) = make_float2(f[0], f[1]);
        else p[0] = f[0];
    } else {
        uint16_t* p = reinterpret_cast<uint16_t*>(base) + off;
        if constexpr (V == 1) p[0] = cvt16<DT == 2>(f[0]);
        else {
            uint32_t w[V / 2];
#pragma unroll
            for (int e = 0; e < V / 2; ++e) w[e] = pack2<DT == 2>(f[2 * e], f[2 * e + 1]);
            if constexpr (V >= 8) {
#pragma unroll
                for (int e = 0; e < V / 8; ++e) reinterpret_cast<uint4*>(p)[e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
            } else if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint32_t*>(p) = w[0];
        }
    }
}

inline int elem_size(int dtype) { return dtype == 0 ? 4 : 2; }
// A launch of 2^32 threads or more along a dimension runs as one of that number modulo 2^32, and no error says so
inline bool launchable(int64_t workgroups, int threads) { return workgroups * threads < (1ll << 32); }

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// V elements as they lie in memory (1 or 2 elements, or 16 bytes), kept packed until they are needed
template <int DT, int V> struct Packed {
    static_assert(V == 1 || V == 2 || V == (DT == 0 ? 4 : 8), "one or two elements, or 16 bytes");
    static constexpr int BYTES = V * (DT == 0 ? 4 : 2);
    typedef typename std::conditional<BYTES == 16, u32x4, typename std::conditional<BYTES == 8, u32x2, typename std::conditional<BYTES == 4, uint32_t, uint16_t>::type>::type>::type T;
    T v;
    __device__ __forceinline__ void load(const void* base, int64_t off) {
        v = *reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + off * (DT == 0 ? 4 : 2));
    }
    __device__ __forceinline__ void clear() {
        if constexpr (BYTES == 16) v = (u32x4){0, 0, 0, 0};
        else if constexpr (BYTES == 8) v = (u32x2){0, 0};
        else v = 0;
    }
    __device__ __forceinline__ void get(float (&f)[V]) const {
        if constexpr (V == 1) {
            if constexpr (DT == 0) f[0] = __uint_as_float(v); else f[0] = xva_glds::ld16<DT == 2>(&v, 0);
        } else if constexpr (DT == 0) {
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = __uint_as_float(v[e]);
        } else if constexpr (V == 2) unpack2<DT == 2>(v, f[0], f[1]);
        else {
#pragma unroll
            for (int e = 0; e < 4; ++e) unpack2<DT == 2>(v[e], f[2 * e], f[2 * e + 1]);
        }
    }
};

// sum over aligned runs of `width` (a power of two, the same in the wave) lanes, in every lane; all lanes active.  Within 16 lanes by DPP: the partner is another
// one of the other half, whose lanes all hold that half's sum by then.
__device__ __forceinline__ float lanes_sum(float v, int width) {
#define XVA_DPP_ADD(ctrl) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, true))
    if (width >= 2) XVA_DPP_ADD(0xB1);            // quad_perm 1 0 3 2
    if (width >= 4) XVA_DPP_ADD(0x4E);            // quad_perm 2 3 0 1
    if (width >= 8) XVA_DPP_ADD(0x141);           // row_half_mirror
    if (width >= 16) XVA_DPP_ADD(0x140);          // row_mirror
#undef XVA_DPP_ADD
    if (width >= 32) v += __shfl_xor(v, 16, 64);
    if (width >= 64) v += __shfl_xor(v, 32, 64);
    return v;
}
}   // namespace xva_seq
