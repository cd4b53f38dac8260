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

// a launch over element type DT and vector width V, both known at run time
template <int DT> struct Elem { static constexpr int size = DT == 0 ? 4 : 2, wide = 16 / size; };   // wide: elements of a 16-byte access
inline int elem_size(int dtype) { return dtype == 0 ? 4 : 2; }
}   // namespace xva_seq
