// Products on FP8 weights: a wave takes 16 weight rows and 16 activation rows, its operands straight from memory, as bf16 (exact).
#include <cstdlib>
#include "fp8.h"

namespace chadq {

typedef __attribute__((ext_vector_type(2))) uint32_t pair_t;

template <bool X8, bool GATED>
__global__ __launch_bounds__(256) void fp8_product_kernel(Fp8Product p) {
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), l16 = lane & 15, kg = lane >> 4;
    const int nwg = blockIdx.y * 64;
    MxTile t = {0, (int)blockIdx.x * 16, p.M - (int)blockIdx.x * 16, 0, 0};
    if (p.offsets) {
        t = MxTiles{p.offsets, p.E, p.M, 16}.find(blockIdx.x);
        if (t.group < 0) {
            if (p.clear_rest) mx_clear(p.y, p.y_bf16, p.N, t, nwg, 64);
            return;
        }
    }
    const int rows = t.rows < 16 ? t.rows : 16, n = nwg + wave * 16 + l16, G = fp8_blocks(p.K), GN = fp8_blocks(p.N);
    const int nr = n < p.N ? n : p.N - 1, m = t.row0 + (l16 < rows ? l16 : rows - 1), xm = p.rows ? p.rows[m] : m;
    constexpr int NB = GATED ? 2 : 1;
    f32x4 acc[NB];
    for (int i = 0; i < NB; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int b = 0; b < G; ++b) {
        f32x4 d[NB];
        for (int i = 0; i < NB; ++i) d[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int j = 0; j < 4; ++j) {
            const int k = b * 128 + j * 32 + kg * 8;
            pair_t w[NB];
            u32x4 xb = {0, 0, 0, 0};
            pair_t x8 = {0, 0};
            for (int i = 0; i < NB; ++i) {
                w[i] = pair_t{0, 0};
                if (k < p.K) w[i] = *reinterpret_cast<const pair_t *>((i ? p.w2 : p.w) + ((size_t)t.group * p.N + nr) * p.K + k);
            }
            if (k < p.K) {
                if (X8) x8 = *reinterpret_cast<const pair_t *>(reinterpret_cast<const uint8_t *>(p.x) + (size_t)xm * p.K + k);
                else xb = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const uint16_t *>(p.x) + (size_t)xm * p.K + k);
            }
            for (int i = 0; i < NB; ++i) {
                const u32x2 lo = fp8_to_bf16(w[i].x), hi = fp8_to_bf16(w[i].y);
                const u32x4 o = {lo.x, lo.y, hi.x, hi.y};
                if (X8) {
                    const u32x2 xl = fp8_to_bf16(x8.x), xh = fp8_to_bf16(x8.y);
                    xb = u32x4{xl.x, xl.y, xh.x, xh.y};
                }
                d[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, o), __builtin_bit_cast(bf16x8, xb), d[i], 0, 0, 0);
            }
        }
        for (int i = 0; i < NB; ++i)
            for (int v = 0; v < 4; ++v) {
                const int c = nwg + wave * 16 + kg * 4 + v;
                float s = (i ? p.w2s : p.ws)[((size_t)t.group * GN + (c < p.N ? c : p.N - 1) / 128) * G + b];
                if (X8) s *= p.xs[(size_t)xm * G + b];
                acc[i][v] += d[i][v] * s;
            }
    }
    if (l16 >= rows) return;
    for (int v = 0; v < 4; ++v) {
        const int c = nwg + wave * 16 + kg * 4 + v;
        if (c < p.N) store_sum(reinterpret_cast<float *>(p.y), (size_t)(t.row0 + l16) * p.N + c, GATED ? silu_mul(acc[0][v], acc[NB - 1][v]) : acc[0][v], p.y_bf16);
    }
}

int fp8_product_launch(const Fp8Product &p, void *workspace, size_t workspace_bytes, hipStream_t st) {
    static const char *const tile = getenv("F8TILE");
    if (!(tile && atoi(tile) >= 100) && fp8_streams(p)) return fp8_stream_launch(p, st);
    if (fp8_tile_ok(p) && !(tile && atoi(tile) < 0)) return fp8_tile_launch(p, tile ? atoi(tile) % 100 : p.M > 256 ? F8_256x256 : p.M > 64 ? F8_256x128 : F8_128x64, st);
    const int64_t tiles = p.offsets ? mx_most_tiles(p.M, p.E, 16) : mx_ceil(p.M, 16), cols = mx_ceil(p.N, 64);
    if (tiles > (1 << 22) || cols > 65535) return fail(CHADQ_ERR_SHAPE, "fp8 product: M=%d N=%d are too many tiles", p.M, p.N);
    const dim3 grid((int)tiles, (int)cols);
    if (p.w2) {
        if (p.xs) hipLaunchKernelGGL((fp8_product_kernel<true, true>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((fp8_product_kernel<false, true>), grid, dim3(256), 0, st, p);
    } else {
        if (p.xs) hipLaunchKernelGGL((fp8_product_kernel<true, false>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((fp8_product_kernel<false, false>), grid, dim3(256), 0, st, p);
    }
    return hip_check(hipGetLastError(), "fp8 product launch");
}

size_t fp8_product_workspace_bytes(int M, int N, int K, bool x_fp8) { return 0; }

}  // namespace chadq
