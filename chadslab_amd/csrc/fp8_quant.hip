// FP8: quantisation (of a block: fp8.h) and its inverse.  Bound by memory, each value read once and written once: 14336 x 4096 fp32 by 128 x 128 46 us, back 42 (294 MB
// each, 6.4 and 7.0 TB/s of which the last-level cache serves a part), 4096 x 4096 bf16 by rows 10.9 (4.7 TB/s), 16 x 4096 2.2 (a launch).
#include "fp8.h"
#include "load8.h"

namespace chadq {

// Rows: 16 lanes to a block, 8 values to a lane.  K is a multiple of 16: pieces of 8 are whole.
template <typename T>
__global__ __launch_bounds__(256) void quantize_fp8_rows_kernel(const T *__restrict__ x, uint8_t *__restrict__ q, float *__restrict__ scale, int64_t rows, int K,
                                                                int G) {
    const int l = threadIdx.x & 15;
    const int64_t blocks = rows * G, stride = (int64_t)gridDim.x * 16;
    for (int64_t b = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4); b < blocks; b += stride) {
        const int64_t row = b / G;
        const int g = (int)(b - row * G), k = g * 128 + l * 8;
        float f[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (k < K) load8<T>(x + row * K + k, f);
        const uint32_t m = absmax8(f);
        const Fp8Scale c(max_of_16(m));
        if (k < K) *reinterpret_cast<u32x2 *>(q + row * K + k) = c.values(f);
        if (l == 0) scale[b] = c.scale;
    }
}

// Weights: a workgroup to a block of 128 x 128, 64 values to a thread: row tid / 16 + 16 i.  first: the launch's first block
template <typename T>
__global__ __launch_bounds__(256) void quantize_fp8_blocks_kernel(const T *__restrict__ x, uint8_t *__restrict__ q, float *__restrict__ scale, int N, int K, int GN,
                                                                  int G, int64_t first) {
    __shared__ uint32_t s_max[4];
    const int64_t b = first + blockIdx.x;
    const int g = (int)(b % G);
    const int64_t rest = b / G;
    const int n0 = (int)(rest % GN) * 128, k = g * 128 + (threadIdx.x & 15) * 8;
    const int64_t base = rest / GN * N;  // first row of the matrix
    float f[8][8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int n = n0 + (threadIdx.x >> 4) + 16 * i;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[i][j] = 0.f;
        if (n < N && k < K) load8<T>(x + (base + n) * K + k, f[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t o = absmax8(f[i]);
        m = o > m ? o : m;
    }
    m = wave_reduce_u32<true, 64>(m);
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) m = s_max[i] > m ? s_max[i] : m;
    const Fp8Scale c(m);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int n = n0 + (threadIdx.x >> 4) + 16 * i;
        if (n < N && k < K) *reinterpret_cast<u32x2 *>(q + (base + n) * K + k) = c.values(f[i]);
    }
    if (threadIdx.x == 0) scale[b] = c.scale;
}

// w = value * scale of its block, one fp32 rounding; 4 values to a lane, so that a wave stores 1 KiB in a row.  high: rows of a block, 1 or 128
__global__ __launch_bounds__(256) void dequant_fp8_kernel(const uint32_t *__restrict__ q, const float *__restrict__ scale, float *__restrict__ w, int64_t rows, int N,
                                                          int K, int GN, int G, int high) {
    const int k4 = K / 4;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const int64_t e = row / N;
        const int n = (int)(row - e * N);
        const float *const s = scale + (e * GN + n / high) * G;
        for (int i = threadIdx.x; i < k4; i += 256) {
            const uint32_t v = q[row * k4 + i];
            const float c = s[i >> 5];
            const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(v, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(v, true);
            __builtin_nontemporal_store(f32x4{a.x * c, a.y * c, b.x * c, b.y * c}, reinterpret_cast<f32x4 *>(w) + row * k4 + i);
        }
    }
}

int quantize_fp8_launch(const void *x, int dtype, uint8_t *q, float *scale, int64_t matrices, int N, int K, bool rows, hipStream_t st) {
    const int G = fp8_blocks(K), GN = fp8_blocks(N);
    const int64_t blocks = rows ? (matrices * N * G + 15) / 16 : matrices * GN * G;
    auto go = [&](auto t) {
        typedef decltype(t) T;
        const T *const from = reinterpret_cast<const T *>(x);
        constexpr int64_t most = 1 << 22;  // workgroups: a launch has fewer than 2^32 threads
        if (rows) hipLaunchKernelGGL(quantize_fp8_rows_kernel<T>, dim3((int)(blocks > 256 * 32 ? 256 * 32 : blocks)), dim3(256), 0, st, from, q, scale, matrices * N, K, G);
        else
            for (int64_t b = 0; b < blocks; b += most)
                hipLaunchKernelGGL(quantize_fp8_blocks_kernel<T>, dim3((int)(blocks - b < most ? blocks - b : most)), dim3(256), 0, st, from, q, scale, N, K, GN, G, b);
    };
    if (dtype == CHADQ_F32) go(float());
    else if (dtype == CHADQ_BF16) go(__bf16());
    else go((_Float16)0);
    return hip_check(hipGetLastError(), "quantize_fp8 launch");
}

int dequant_fp8_launch(const uint8_t *q, const float *scale, float *w, int64_t matrices, int N, int K, bool by_row, hipStream_t st) {
    const int64_t rows = matrices * N;
    hipLaunchKernelGGL(dequant_fp8_kernel, dim3((int)(rows < 65536 ? rows : 65536)), dim3(256), 0, st, reinterpret_cast<const uint32_t *>(q), scale, w, rows, N, K,
                       by_row ? N : fp8_blocks(N), fp8_blocks(K), by_row ? 1 : 128);
    return hip_check(hipGetLastError(), "dequant_fp8 launch");
}

}  // namespace chadq
