// Products of at most 16 rows (of a group) on MXFP4 weights: y[m,n] = sum_k x[m,k] value(w[n,k]) 2^(e[n,k/32] - 127), x bf16 or MXFP4, one
// matrix or one per group of rows.  HBM-bound: every weight is read once per tile of 16 rows.
//
// A workgroup's W waves share NT blocks of at most 16 weight rows and split K among them, 128 k (a unit: four scale blocks, one to each
// 16 lanes) at a time, D units of a wave one behind the other, their weights requested a round (D units of every wave) ahead.  Weights go from memory
// straight into the operand registers, 16 bytes = one scale block per lane; the activations wait in LDS, requested before the first weights, zeros behind
// K, where a lane past the end of its weight row reads that row's last block again (what is NaN there makes the row's result NaN in any case).
// bf16 activations: the codes become bf16 with their scale, exactly, by one conversion per pair, and v_mfma_f32_16x16x32_bf16 sums in fp32.
// MXFP4 activations: both operands go to v_mfma_scale_f32_16x16x128_f8f6f4 as they are.  The weights are the first operand, so that a lane ends up
// with four consecutive n of one activation row.  The waves' sums meet in LDS, added in their order.
#include "mx.h"

namespace chadq {

// What the first requests need comes first in the arguments, where it arrives in registers with the wave.
// RT: weight rows of a block in use (<= 16); KU: units of a chunk of activations, whole rounds; inv: 65536 / KiB of a chunk's row, rounded up
// GATED: every second block is of w2, of the same rows as the block of w before it
template <bool X4, bool GATED, bool GROUPED, int NT, int W, int D>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(4))) void mx_stream_kernel(
    const uint8_t *__restrict__ x, const uint8_t *__restrict__ w, const uint8_t *__restrict__ ws, int K, int N, int M, int RT, int KU, int inv, void *y, int y_bf16,
    const uint8_t *__restrict__ xs, const int32_t *__restrict__ offsets, int E, bool clear_rest, const int32_t *__restrict__ xrows, const uint8_t *__restrict__ w2,
    const uint8_t *__restrict__ w2s) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, kg = lane >> 4;
    constexpr int NO = GATED ? NT / 2 : NT;  // blocks of results
    const int n0 = blockIdx.y * (NO * RT), G = K >> 5, rounds = ((G + 3) / 4 + W * D - 1) / (W * D);
    MxTile t = {0, (int)blockIdx.x * 16, M - (int)blockIdx.x * 16, 0, 0};
    if constexpr (GROUPED) {
        t = MxTiles{offsets, E, M, 16}.find(blockIdx.x);
        if (t.group < 0) {
            if (clear_rest) mx_clear(y, y_bf16, N, t, n0, NO * RT);
            return;
        }
    }
    const int rows = t.rows < 16 ? t.rows : 16;

    // ---- activations.  A chunk: rows of KU units, 16 bytes apart beyond that (16 rows then cover the banks)
    constexpr int UB = X4 ? 64 : 256;  // bytes of a unit
    const int pitch = KU * UB + 16, per = KU * UB / 1024;
    const int xrow = X4 ? K >> 1 : K * 2;  // bytes of a row
    auto stage = [&](int u0) {  // 1 KiB of a row per request; past a row's end nothing is read and zeros arrive
        for (int i = wave; i < rows * per; i += W) {
            const int r = (i * inv) >> 16, b = (i - r * per) * 1024, at = u0 * UB + b + lane * 16;
            const int src = GATED ? __builtin_amdgcn_readfirstlane(xrows[t.row0 + r]) : t.row0 + r;
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(x) + (size_t)src * xrow, 0, xrow, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void *)(lds + r * pitch + b), 16, at < xrow ? (uint32_t)at : 0x80000000u, 0, 0, 0);
        }
    };
    stage(0);

    // ---- weights
    const uint8_t *wrow[NT], *srow[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        int n = n0 + (GATED ? i / 2 : i) * RT + (l16 < RT ? l16 : RT - 1);
        n = n < N ? n : N - 1;
        const size_t r = (size_t)t.group * N + n;
        wrow[i] = (GATED && i % 2 ? w2 : w) + r * (size_t)(K >> 1);
        srow[i] = (GATED && i % 2 ? w2s : ws) + r * (size_t)G;
    }
    const int xm = l16 < rows ? l16 : rows - 1;  // the lane's activation row (one of the tile's, where it has fewer)
    const uint8_t *const xsrow = X4 ? xs + (size_t)(t.row0 + xm) * G : nullptr;
    u32x4 q[D][NT];
    uint32_t s[NT], sx;  // scales of a round's D units: those of unit kg of them
    auto load_w = [&](int round, int d) {
        int b = ((round * W + wave) * D + d) * 4 + kg;
        b = b < G ? b : G - 1;
#pragma unroll
        for (int i = 0; i < NT; ++i) q[d][i] = load_nt_b128(wrow[i] + (size_t)b * 16);
    };
    auto load_s = [&](int round) {
        const int at = ((round * W + wave) * D + (kg < D ? kg : D - 1)) * 4;
#pragma unroll
        for (int i = 0; i < NT; ++i) s[i] = (uint32_t)load_scales<4>(srow[i], at, G);
        if constexpr (X4) sx = (uint32_t)load_scales<4>(xsrow, at, G);
    };
    // unit d's four scales are in the lanes of group d; every lane wants that of its own block: byte kg
    auto scales_of = [&](uint32_t v, uint32_t out[D]) {
        uint32_t a = v, b = v;
        if constexpr (D > 1) {
            const auto p16 = __builtin_amdgcn_permlane16_swap(v, v, false, false);  // groups 0 0 2 2 and 1 1 3 3
            a = p16[0];
            b = p16[1];
        }
        const auto pa = __builtin_amdgcn_permlane32_swap(a, a, false, false);
        out[0] = pa[0] >> (8 * kg);
        if constexpr (D > 1) {
            const auto pb = __builtin_amdgcn_permlane32_swap(b, b, false, false);
            out[1] = pb[0] >> (8 * kg);
            if constexpr (D > 2) {
                out[2] = pa[1] >> (8 * kg);
                out[3] = pb[1] >> (8 * kg);
            }
        }
    };
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    load_s(0);
#pragma unroll
    for (int d = 0; d < D; ++d) load_w(0, d);
    __builtin_amdgcn_sched_barrier(0);

    f32x4 acc[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const uint8_t *const xl = lds + xm * pitch + (X4 ? kg * 16 : kg * 64) + wave * D * UB;

    if (G >= 4) wait_vmcnt<NT + X4 + D * NT>();  // what has been requested since the activations
    else wait_vmcnt<0>();
    wg_barrier();
    int at = 0;  // of the round in its chunk
    auto turn = [&](int round, bool more) {
        const uint8_t *const xr = xl + at * (W * D * UB);
        uint32_t sc[NT][D], sxc[D];
#pragma unroll
        for (int i = 0; i < NT; ++i) scales_of(s[i], sc[i]);
        if constexpr (X4) scales_of(sx, sxc);
        if (more) load_s(round + 1);
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if constexpr (X4) {
                const i32x8 xo = mx_operand(*reinterpret_cast<const u32x4 *>(xr + d * UB));
#pragma unroll
                for (int i = 0; i < NT; ++i)
                    acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(q[d][i]), xo, acc[i], 4, 4, 0, (int)sc[i][d], 0, (int)sxc[d]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bf16x8 xo = *reinterpret_cast<const bf16x8 *>(xr + d * UB + j * 16);
#pragma unroll
                    for (int i = 0; i < NT; ++i)
                        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(dequant8_mx(q[d][i][j], mx_scale(sc[i][d] & 255u)), xo, acc[i], 0, 0, 0);
                }
            }
            if (more) load_w(round + 1, d);
            __builtin_amdgcn_sched_barrier(0);
        }
        ++at;
    };
    int round = 0;
    for (; round + 1 < rounds; ++round) {
        turn(round, true);
        if (at * (W * D) == KU) {  // the next chunk
            wg_barrier();
            stage((round + 1) * (W * D));
            wait_vmcnt<0>();
            wg_barrier();
            at = 0;
        }
    }
    turn(round, false);

    // ---- the waves' sums: [wave][block][lane] of four n each
    wg_barrier();
    f32x4 *const part = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
    for (int i = 0; i < NT; ++i) part[(wave * NT + i) * 64 + lane] = acc[i];
    wg_barrier();
    auto sum = [&](int i) {
        f32x4 v = part[i];
#pragma unroll
        for (int w = 1; w < W; ++w) v += part[w * NT * 64 + i];
        return v;
    };
    for (int i = tid; i < NO * 64; i += 64 * W) {
        const int m = i & 15, b = i / 64, r = (i & 63) / 16 * 4, e = (GATED ? 2 * b : b) * 64 + (i & 63);
        if (m >= rows || r >= RT) continue;
        f32x4 v = sum(e);
        if constexpr (GATED) {
            const f32x4 u = sum(e + 64);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = silu_mul(v[j], u[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = n0 + b * RT + r + j;
            if (r + j < RT && n < N) store_sum(reinterpret_cast<float *>(y), (size_t)(t.row0 + m) * N + n, v[j], y_bf16);
        }
    }
}

template <bool X4, bool GATED, bool GROUPED, int NT, int W, int D>
static int launch(const MxProduct &p, int RT, hipStream_t st) {
    constexpr int NO = GATED ? NT / 2 : NT, UB = X4 ? 64 : 256;
    const int U = (p.K + 127) / 128, round = W * D, rounds = (U + round - 1) / round, rows = p.M < 16 ? p.M : 16;
    const int most = (W == 8 ? 73728 : 147456) / (rows * round * UB), chunk = most < 1 ? 1 : most > rounds ? rounds : most;  // rounds of a chunk
    const int ku = chunk * round;
    static_assert(W * D * UB % 1024 == 0, "a request fills a KiB of a row");
    const size_t part = (size_t)W * NT * 1024, xb = (size_t)rows * (ku * UB + 16), lds = part > xb ? part : xb;
    if (lds > 163840) return fail(CHADQ_ERR_SHAPE, "mxfp4 product: %zu bytes of LDS", lds);
    const int64_t tiles = p.offsets ? mx_most_tiles(p.M, p.E, 16) : (p.M + 15) / 16, cols = ((int64_t)p.N + NO * RT - 1) / (NO * RT);
    if (tiles > INT32_MAX || cols > 65535) return fail(CHADQ_ERR_SHAPE, "mxfp4 product: M=%d N=%d are too many tiles", p.M, p.N);
    static std::atomic<bool> set[64];  // more LDS than the default limit: once per device
    int dev = 0;
    CHADQ_HIP(hipGetDevice(&dev));
    if (dev >= 64 || !set[dev].load()) {
        CHADQ_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(&mx_stream_kernel<X4, GATED, GROUPED, NT, W, D>), hipFuncAttributeMaxDynamicSharedMemorySize, 163840));
        if (dev < 64) set[dev].store(true);
    }
    hipLaunchKernelGGL((mx_stream_kernel<X4, GATED, GROUPED, NT, W, D>), dim3((int)tiles, (int)cols), dim3(64 * W), lds, st,
                       reinterpret_cast<const uint8_t *>(p.x), p.w, p.ws, p.K, p.N, p.M, RT, ku, 65536 / (ku * UB / 1024) + 1, p.y, (int)p.y_bf16, p.xs, p.offsets, p.E,
                       p.clear_rest, p.rows, p.w2, p.w2s);
    return hip_check(hipGetLastError(), "mxfp4 product launch");
}

template <bool X4, bool GATED, bool GROUPED, int NT>
static int launch_waves(const MxProduct &p, int RT, hipStream_t st) {
    const int U = (p.K + 127) / 128;
    // 16 waves, one workgroup to a compute unit, where two workgroups' activations would not fit beside each other (or are read twice)
    if ((p.offsets ? 16 : p.M) > 8) return launch<X4, GATED, GROUPED, NT, 16, 2>(p, RT, st);
    if constexpr (!X4)
        if (U <= 8) return launch<X4, GATED, GROUPED, NT, 8, 1>(p, RT, st);
    if constexpr (NT < 4)
        if (U > 16) return launch<X4, GATED, GROUPED, NT, 8, 4>(p, RT, st);
    return launch<X4, GATED, GROUPED, NT, 8, 2>(p, RT, st);
}

template <bool X4, bool GATED, bool GROUPED>
static int launch_blocks(const MxProduct &p, hipStream_t st) {
    constexpr int PAIR = GATED ? 2 : 1;  // blocks of a result block
    if constexpr (GROUPED) {
        return launch_waves<X4, GATED, GROUPED, 2 * PAIR>(p, 16, st);
    } else {
        // As many rows to a workgroup as give every compute unit the same number of them (one, or two of 8 waves)
        const int most = p.M > 8 && !X4 ? 64 : 32, rounds = (p.N + 256 * most - 1) / (256 * most), rows = (p.N + 256 * rounds - 1) / (256 * rounds);
        const int blocks = (rows + 15) / 16;
        if (blocks <= 1) return launch_waves<X4, GATED, GROUPED, 1>(p, rows, st);
        if constexpr (!X4)
            if (blocks > 2) return launch_waves<X4, GATED, GROUPED, 4>(p, (rows + 3) / 4, st);
        return launch_waves<X4, GATED, GROUPED, 2>(p, (rows + 1) / 2, st);
    }
}

int mx_stream_launch(const MxProduct &p, hipStream_t st) {
    if (p.w2) return launch_blocks<false, true, true>(p, st);
    if (p.offsets) return p.xs ? launch_blocks<true, false, true>(p, st) : launch_blocks<false, false, true>(p, st);
    return p.xs ? launch_blocks<true, false, false>(p, st) : launch_blocks<false, false, false>(p, st);
}

size_t mx_product_workspace_bytes(int, int, int, bool) { return 0; }

int mx_product_launch(const MxProduct &p, void *, size_t, hipStream_t st) {
    const int per = p.offsets ? (p.M + p.E - 1) / p.E : p.M;
    return per > 16 && mx_tile_ok(p) ? mx_tile_launch(p, st) : mx_stream_launch(p, st);
}

}  // namespace chadq
