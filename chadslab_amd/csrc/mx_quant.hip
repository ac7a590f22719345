// MXFP4: quantisation and its inverse.  Per block of 32 values along K:  e = clamp(floor(log2 max|x|) - 2 + 127, 0, 254),
// code = the nearest e2m1 to x / 2^(e - 127), ties to the even one, what lies beyond 6 to 6; a block that holds a NaN or an
// infinity gets e = 255 and codes of 0.  The division by a power of two is exact, so there is nothing to round but the code.
//
// Both are bound by the bytes they move.  Over inputs and results that do not fit the 256 MB cache: quantising 14336 x 4096 fp32 46.6 us = 5.7 TB/s, seven eighths of
// it read, 4096 x 4096 bf16 9.1 us = 4.7 TB/s, and dequantising 14336 x 4096 55.9 us = 4.8 TB/s, seven eighths written (a copy of 1 GiB moves 5.2 TB/s, read and written, filling it
// 6.8); with results that the cache holds 8.5 and 45.5 us.  16 x 4096: 3.2 us, a launch and one trip to memory.
#include "mx.h"

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

// Four lanes to a block, 8 values to a lane: a lane stores one word of codes, and two exchanges inside the quad give the block's largest magnitude.
// Rows do not matter, K is a multiple of 32.
template <typename T>
__global__ __launch_bounds__(256) void quantize_mxfp4_kernel(const T *__restrict__ x, uint32_t *__restrict__ codes, uint8_t *__restrict__ scale,
                                                             int64_t n8) {
    const int64_t stride = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n8; i += stride) {  // n8 is a multiple of 4: quads stay whole
        float f[8];
        load8<T>(x + i * 8, f);
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t b = __float_as_uint(f[j]) & 0x7FFFFFFFu;  // as integers: a NaN is larger than infinity
            m = b > m ? b : m;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const uint32_t o = (uint32_t)(s ? __builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false)    // quad_perm [2,3,0,1]
                                            : __builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));  // quad_perm [1,0,3,2]
            m = o > m ? o : m;
        }
        const uint32_t e = m >> 23, byte = e == 255 ? 255 : e > 2 ? e - 2 : 0;
        const float s = mx_scale(byte);
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[0], f[1], s, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[2], f[3], s, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[4], f[5], s, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[6], f[7], s, 3);
        codes[i] = byte == 255 ? 0u : c;
        if ((i & 3) == 0) scale[i >> 2] = (uint8_t)byte;
    }
}

// w[i] = value(code i) * scale of its block as fp32, exact (beyond fp32's range: infinity); 4 codes to a lane, so that a wave stores 1 KiB in a row, four
// times in flight.  The stores go past the caches: 14336 x 4096, into a result that the last cache holds, 65 -> 45 us with both.
__global__ __launch_bounds__(256) void dequant_mxfp4_kernel(const uint16_t *__restrict__ codes, const uint8_t *__restrict__ scale,
                                                            float *__restrict__ w, int64_t n4) {
    const int64_t stride = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += 4 * stride) {
        uint32_t c[4], s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t at = i + j * stride < n4 ? i + j * stride : i;
            c[j] = codes[at];
            s[j] = scale[at >> 3];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i + j * stride >= n4) break;
            const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[j], mx_scale(s[j]), 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[j], mx_scale(s[j]), 1);
            __builtin_nontemporal_store(f32x4{a.x, a.y, b.x, b.y}, reinterpret_cast<f32x4 *>(w) + i + j * stride);
        }
    }
}

static int grid_for(int64_t items) {
    const int64_t b = (items + 255) / 256;
    return b < 1 ? 1 : b > 256 * 32 ? 256 * 32 : (int)b;
}

int quantize_mxfp4_launch(const void *x, int dtype, uint8_t *codes, uint8_t *scale, int64_t rows, int K, hipStream_t st) {
    const int64_t n8 = rows * (K / 8);
    uint32_t *const c = reinterpret_cast<uint32_t *>(codes);
    if (dtype == CHADQ_F32) hipLaunchKernelGGL(quantize_mxfp4_kernel<float>, dim3(grid_for(n8)), dim3(256), 0, st, reinterpret_cast<const float *>(x), c, scale, n8);
    else if (dtype == CHADQ_BF16) hipLaunchKernelGGL(quantize_mxfp4_kernel<__bf16>, dim3(grid_for(n8)), dim3(256), 0, st, reinterpret_cast<const __bf16 *>(x), c, scale, n8);
    else hipLaunchKernelGGL(quantize_mxfp4_kernel<_Float16>, dim3(grid_for(n8)), dim3(256), 0, st, reinterpret_cast<const _Float16 *>(x), c, scale, n8);
    return hip_check(hipGetLastError(), "quantize_mxfp4 launch");
}

int dequant_mxfp4_launch(const uint8_t *codes, const uint8_t *scale, float *w, int64_t rows, int K, hipStream_t st) {
    const int64_t n4 = rows * (K / 4);
    hipLaunchKernelGGL(dequant_mxfp4_kernel, dim3(grid_for((n4 + 3) / 4)), dim3(256), 0, st, reinterpret_cast<const uint16_t *>(codes), scale, w, n4);
    return hip_check(hipGetLastError(), "dequant_mxfp4 launch");
}

}  // namespace chadq
