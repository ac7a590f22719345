// 8 consecutive values of any of the three types that quantisers take.
#pragma once
#include "chadq_common.h"

namespace chadq {

// the bits of 8 consecutive values as fp32
template <typename T>
__device__ __forceinline__ void load8(const T *p, float f[8]);
template <>
__device__ __forceinline__ void load8<float>(const float *p, float f[8]) {
    const f32x4 a = reinterpret_cast<const f32x4 *>(p)[0], b = reinterpret_cast<const f32x4 *>(p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = a[i];
        f[4 + i] = b[i];
    }
}
template <>
__device__ __forceinline__ void load8<__bf16>(const __bf16 *p, float f[8]) {
    const u32x4 v = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(v[i] << 16);
        f[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
    }
}
template <>
__device__ __forceinline__ void load8<_Float16>(const _Float16 *p, float f[8]) {
    const u32x4 v = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f16x2 h = as_f16x2(v[i]);
        f[2 * i] = (float)h.x;
        f[2 * i + 1] = (float)h.y;
    }
}

}  // namespace chadq
