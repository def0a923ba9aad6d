// Elements of feature rows in registers: 8 at a time, f32 / bf16 / f16, any alignment (the row of an odd width starts at any element), the end of a row by element.
#pragma once
#include "common.h"

namespace {

template <int DT> struct Elem;
template <> struct Elem<W3D_DTYPE_F32> { static constexpr int B = 4; };
template <> struct Elem<W3D_DTYPE_BF16> { static constexpr int B = 2; };
template <> struct Elem<W3D_DTYPE_F16> { static constexpr int B = 2; };
template <> struct Elem<W3D_DTYPE_FP8_E4M3> { static constexpr int B = 1; };

__device__ __forceinline__ float f16_to_f32(uint16_t b) { _Float16 h; __builtin_memcpy(&h, &b, 2); return (float)h; }
__device__ __forceinline__ uint16_t f32_to_f16(float f) { _Float16 h = (_Float16)f; uint16_t b; __builtin_memcpy(&b, &h, 2); return b; }

template <int DT>
__device__ __forceinline__ float load1(const void *p) {
    if (DT == W3D_DTYPE_F32) { float v; __builtin_memcpy(&v, p, 4); return v; }
    uint16_t b; __builtin_memcpy(&b, p, 2);
    return DT == W3D_DTYPE_BF16 ? bf16_to_f32(b) : f16_to_f32(b);
}
template <int DT>
__device__ __forceinline__ void store1(void *p, float v) {
    if (DT == W3D_DTYPE_F32) { __builtin_memcpy(p, &v, 4); return; }
    const uint16_t b = DT == W3D_DTYPE_BF16 ? f32_to_bf16(v) : f32_to_f16(v);
    __builtin_memcpy(p, &b, 2);
}

// elements [0, n) of p (n may exceed 8 or be <= 0), zero beyond: the vector load is a plain one of any alignment (global memory takes dword loads at any byte)
template <int DT>
__device__ __forceinline__ void load8(const void *p, int n, float (&v)[8]) {
    if (n >= 8) {
        if (DT == W3D_DTYPE_F32) { __builtin_memcpy(v, p, 32); return; }
        uint32_t w[4];
        __builtin_memcpy(w, p, 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (DT == W3D_DTYPE_BF16) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
            else { v[2 * i] = f16_to_f32((uint16_t)w[i]); v[2 * i + 1] = f16_to_f32((uint16_t)(w[i] >> 16)); }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? load1<DT>((const char *)p + i * Elem<DT>::B) : 0.f;
}
template <int DT>
__device__ __forceinline__ void store8(void *p, int n, const float (&v)[8]) {
    if (n >= 8) {
        if (DT == W3D_DTYPE_F32) { __builtin_memcpy(p, v, 32); return; }
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint16_t a = DT == W3D_DTYPE_BF16 ? f32_to_bf16(v[2 * i]) : f32_to_f16(v[2 * i]);
            const uint16_t b = DT == W3D_DTYPE_BF16 ? f32_to_bf16(v[2 * i + 1]) : f32_to_f16(v[2 * i + 1]);
            w[i] = (uint32_t)a | ((uint32_t)b << 16);
        }
        __builtin_memcpy(p, w, 16);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) store1<DT>((char *)p + i * Elem<DT>::B, v[i]);
}

}  // namespace
