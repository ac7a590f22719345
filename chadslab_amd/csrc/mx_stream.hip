// Products of few rows on MXFP4 weights: y[m,n] = sum_k x[m,k] value(w[n,k]) 2^(e[n,k/32] - 127), x bf16 or MXFP4, one matrix or
// (groups) one per run of rows.  HBM-bound: every weight is read once per tile of 16 MT rows.
//
// A workgroup's W waves share NT blocks of at most 16 weight rows and split K among them, 128 k (a unit: four scale blocks, one to each
// 16 lanes) at a time.  Weights go from memory straight into the operand registers, 16 bytes = one scale block per lane; the
// activations wait in LDS, zeros behind K, where a lane past the end of its weight row reads that row's last block again (what is
// NaN there makes the row's result NaN in any case).  bf16 activations: the codes become bf16 with their scale, exactly, by one conversion per pair, and
// v_mfma_f32_16x16x32_bf16 sums in fp32.  MXFP4 activations: both operands go to v_mfma_scale_f32_16x16x128_f8f6f4 as they are.  The weights
// are the first operand, so that a lane ends up with four consecutive n of one activation row.  The waves' sums meet in LDS, added in their order.
#include "mx.h"

namespace chadq {

// RT: weight rows of a block in use (<= 16); KU: units of a chunk of activations, a multiple of W * DEPTH
// GATED: every second block is of w2, of the same rows as the block of w before it
template <bool X4, bool GATED, int MT, int NT, int W, int DEPTH>
__global__ __launch_bounds__(64 * W) void mx_stream_kernel(MxProduct p, int RT, int KU) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, kg = lane >> 4;
    constexpr int NO = GATED ? NT / 2 : NT;  // blocks of results
    const int n0 = blockIdx.y * (NO * RT), G = p.K >> 5, U = (G + 3) >> 2;
    MxTile t = {0, (int)blockIdx.x * (16 * MT), p.M - (int)blockIdx.x * (16 * MT), 0, 0};
    if (p.offsets) {
        t = MxTiles{p.offsets, p.E, p.M, 16 * MT}.find(blockIdx.x);
        if (t.group < 0) {
            if (p.clear_rest) mx_clear(p, t, n0, NO * RT);
            return;
        }
    }
    const int rows = t.rows < 16 * MT ? t.rows : 16 * MT;
    const uint8_t *wrow[NT], *srow[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        int n = n0 + (GATED ? i / 2 : i) * RT + (l16 < RT ? l16 : RT - 1);
        n = n < p.N ? n : p.N - 1;
        const size_t r = (size_t)t.group * p.N + n;
        wrow[i] = (GATED && i % 2 ? p.w2 : p.w) + r * (size_t)(p.K >> 1);
        srow[i] = (GATED && i % 2 ? p.w2s : p.ws) + r * (size_t)G;
    }
    u32x4 q[DEPTH][NT];
    uint32_t s[DEPTH][NT];
    auto load = [&](int u, int d) {
        int b = 4 * u + kg;
        b = b < G ? b : G - 1;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            q[d][i] = load_nt_b128(wrow[i] + (size_t)b * 16);
            s[d][i] = srow[i][b];
        }
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(wave + d * W, d);

    // chunk: rows of KU units, 16 bytes apart beyond that (16 rows then cover the banks); behind them the scales of MXFP4 rows
    constexpr int UB = X4 ? 64 : 256;  // bytes of a unit
    const int pitch = KU * UB + 16, spitch = KU * 4 + 4;
    uint8_t *const xsl = lds + rows * pitch;
    const int xrow = X4 ? p.K >> 1 : p.K * 2;  // bytes of a row
    auto stage = [&](int u0) {
        const int per = KU * UB / 16;
        for (int i = tid; i < rows * per; i += 64 * W) {
            const int r = i / per, b = (i % per) * 16, at = u0 * UB + b;
            u32x4 v = {0u, 0u, 0u, 0u};
            if (at < xrow) {
                const int src = p.rows ? p.rows[t.row0 + r] : t.row0 + r;
                v = *reinterpret_cast<const u32x4 *>(reinterpret_cast<const uint8_t *>(p.x) + (size_t)src * xrow + at);
            }
            *reinterpret_cast<u32x4 *>(lds + r * pitch + b) = v;
        }
        if constexpr (X4)
            for (int i = tid; i < rows * KU * 4; i += 64 * W) {
                const int r = i / (KU * 4), b = i % (KU * 4), at = u0 * 4 + b;
                xsl[r * spitch + b] = at < G ? p.xs[(size_t)(t.row0 + r) * G + at] : (uint8_t)0;
            }
    };

    f32x4 acc[MT][NT];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    int xm[MT];  // the lane's activation row in each row block (one of the tile's, where the block has fewer)
#pragma unroll
    for (int a = 0; a < MT; ++a) xm[a] = a * 16 + l16 < rows ? a * 16 + l16 : rows - 1;

    for (int u0 = 0; u0 < U; u0 += KU) {
        if (u0) __syncthreads();
        stage(u0);
        __syncthreads();
        const int end = U - u0 < KU ? U - u0 : KU;
        for (int i = wave; i < end; i += W * DEPTH) {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                const int v = i + d * W;
                if (v < end) {
                    if constexpr (X4) {
                        i32x8 xo[MT];
                        int xsc[MT];
#pragma unroll
                        for (int a = 0; a < MT; ++a) {
                            xo[a] = mx_operand(*reinterpret_cast<const u32x4 *>(lds + xm[a] * pitch + v * 64 + kg * 16));
                            xsc[a] = xsl[xm[a] * spitch + v * 4 + kg];
                        }
#pragma unroll
                        for (int b = 0; b < NT; ++b)
#pragma unroll
                            for (int a = 0; a < MT; ++a)
                                acc[a][b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(q[d][b]), xo[a], acc[a][b], 4, 4, 0, (int)s[d][b], 0, xsc[a]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            bf16x8 xo[MT];
#pragma unroll
                            for (int a = 0; a < MT; ++a) xo[a] = *reinterpret_cast<const bf16x8 *>(lds + xm[a] * pitch + v * 256 + kg * 64 + j * 16);
#pragma unroll
                            for (int b = 0; b < NT; ++b) {
                                const bf16x8 wo = dequant8_mx(q[d][b][j], mx_scale(s[d][b]));
#pragma unroll
                                for (int a = 0; a < MT; ++a) acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wo, xo[a], acc[a][b], 0, 0, 0);
                            }
                        }
                    }
                }
                load(u0 + v + W * DEPTH, d);
            }
        }
    }

    // ---- the waves' sums: [wave][block][lane] of four n each
    __syncthreads();
    f32x4 *const part = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int b = 0; b < NT; ++b) part[(wave * MT * NT + a * NT + b) * 64 + lane] = acc[a][b];
    __syncthreads();
    auto sum = [&](int i) {
        f32x4 v = part[i];
        for (int w = 1; w < W; ++w) v += part[w * MT * NT * 64 + i];
        return v;
    };
    for (int i = tid; i < MT * NO * 64; i += 64 * W) {
        const int m = i / (64 * NO) * 16 + (i & 15), b = i / 64 % NO, r = (i & 63) / 16 * 4;
        const int at = (i / (64 * NO) * NT + (GATED ? 2 * b : b)) * 64 + (i & 63);
        f32x4 v = sum(at);
        if constexpr (GATED) {
            const f32x4 u = sum(at + 64);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = silu_mul(v[j], u[j]);
        }
        if (m >= rows) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + b * RT + r + j;
            if (r + j < RT && n < p.N) store_sum(reinterpret_cast<float *>(p.y), (size_t)(t.row0 + m) * p.N + n, v[j], p.y_bf16);
        }
    }
}

template <bool X4, bool GATED, int MT>
static int launch(const MxProduct &p, hipStream_t st) {
    constexpr int NT = 2, W = 8, DEPTH = 4 / MT, RT = 16, NO = GATED ? NT / 2 : NT;
    const int U = (p.K + 127) / 128, step = W * DEPTH;
    const int rows = p.M < 16 * MT ? p.M : 16 * MT, unit = rows * (X4 ? 68 : 256);
    int ku = (65536 / unit) / step * step;  // units of a chunk: 64 KiB of activations, whole rounds of the waves
    const int all = (U + step - 1) / step * step;
    ku = ku < step ? step : ku > all ? all : ku;
    const size_t part = (size_t)W * MT * NT * 1024, chunk = (size_t)rows * (ku * (X4 ? 64 : 256) + 16 + (X4 ? ku * 4 + 4 : 0));
    const size_t lds = part > chunk ? part : chunk;
    const int64_t tiles = p.offsets ? mx_most_tiles(p.M, p.E, 16 * MT) : (p.M + 16 * MT - 1) / (16 * MT);
    const int64_t cols = ((int64_t)p.N + NO * RT - 1) / (NO * RT);
    if (tiles > INT32_MAX || cols > 65535) return fail(CHADQ_ERR_SHAPE, "mxfp4 product: M=%d N=%d are too many tiles", p.M, p.N);
    static std::atomic<bool> set[64];  // more LDS than the default limit: once per device
    int dev = 0;
    CHADQ_HIP(hipGetDevice(&dev));
    if (dev >= 64 || !set[dev].load()) {
        CHADQ_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(&mx_stream_kernel<X4, GATED, MT, NT, W, DEPTH>), hipFuncAttributeMaxDynamicSharedMemorySize, 163840));
        if (dev < 64) set[dev].store(true);
    }
    hipLaunchKernelGGL((mx_stream_kernel<X4, GATED, MT, NT, W, DEPTH>), dim3((int)tiles, (int)cols), dim3(64 * W), lds, st, p, RT, ku);
    return hip_check(hipGetLastError(), "mxfp4 product launch");
}

template <bool X4, bool GATED>
static int launch_rows(const MxProduct &p, hipStream_t st) {
    const int per = p.offsets ? (p.M + p.E - 1) / p.E : p.M;
    return per <= 16 ? launch<X4, GATED, 1>(p, st) : per <= 32 ? launch<X4, GATED, 2>(p, st) : launch<X4, GATED, 4>(p, st);
}

int mx_stream_launch(const MxProduct &p, hipStream_t st) {
    if (p.w2) return launch_rows<false, true>(p, st);
    return p.xs ? launch_rows<true, false>(p, st) : launch_rows<false, false>(p, st);
}

size_t mx_product_workspace_bytes(int, int, int, bool) { return 0; }

int mx_product_launch(const MxProduct &p, void *, size_t, hipStream_t st) {
    const int per = p.offsets ? (p.M + p.E - 1) / p.E : p.M;
    return per > 64 && mx_tile_ok(p) ? mx_tile_launch(p, st) : mx_stream_launch(p, st);
}

}  // namespace chadq
