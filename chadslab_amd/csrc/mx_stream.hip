// Products of at most 16 rows (of a group) on MXFP4 weights: y[m,n] = sum_k x[m,k] value(w[n,k]) 2^(e[n,k/32] - 127), x bf16 or MXFP4, one
// matrix or one per group of rows.  HBM-bound: every weight is read once per tile of 8 MT rows.
//
// A wave works on 8 weight rows, 256 k (a unit: eight scale blocks) at a time: one load instruction brings 128 consecutive bytes of each row, 16 bytes = one
// block per lane, straight into the operand registers.  The matrix instruction has 16 weight rows and 4 blocks instead; so each row takes two of its
// rows, with blocks 0-3 and 4-7, and the activations take two columns each, row m's blocks 0-3 in column m and 4-7 in column 8 + m: of the result
// the (even row, column m) and (odd row, column 8 + m) are wanted and added at the end.  (16 rows x 64 bytes per load instead, no half of the result
// thrown away: 1 x 14336 x 4096 9.0 instead of 7.8 us; the matrix cores have time to spare, the 64-byte pieces cost memory.)  MT = 2: rows 8-15 by a
// second instruction.
//   bf16 x   the codes become bf16 with their scale, exactly, one conversion per pair; v_mfma_f32_16x16x32_bf16 sums in fp32
//   MXFP4 x  both operands go to v_mfma_scale_f32_16x16x128_f8f6f4 as they are
// A workgroup's eight waves are S = 8 / WK side by side in n and WK along K.  A round is D units of each wave; its weights are requested a round ahead.
// The activations wait in LDS, a chunk of rounds at a time, requested before the first weights; behind K they are zeros, and a lane past
// the end of its weight row reads that row's last codes again, with a scale of 2^-127.  Scales: a round's 8 D bytes
// of a row are loaded by the row's eight lanes together and go through LDS, where each lane picks its blocks'.
//
// Measured over rotating weights, bf16 x: 1 x 2048 x 2048 3.3 us (a launch alone 1.7), 1 x 14336 x 4096 7.5 us = 4.2 TB/s, 6 x 11008 x 4096 6.9 us, 16 x
// 14336 x 4096 11.4 us (MXFP4 x: 8.0), 32 rows by 8 matrices of 14336 x 4096 49.8 us = 5.0 TB/s.  Few rows: what is left of the time is the launch and the first
// round's trip to memory.  16 rows: the activations, 128 KiB to each of 256 workgroups through L2 (read there by the lanes themselves instead: 16.7 for 12.3 us).
#include "mx.h"

namespace chadq {

constexpr int MXS_W = 8;  // waves
constexpr int kStreamCols = 65535;  // workgroups along n: a grid's second dimension

// What the first requests need comes first in the arguments, where it arrives in registers with the wave.
// RT: weight rows of a wave in use (<= 8); wk: log2 WK; chunk: rounds of a chunk of activations; inv: 65536 / KiB of its rows, rounded up
// GATED: gate rows w and up rows w2, bf16(silu(gate) up)
template <bool X4, bool GATED, bool GROUPED, int MT, int D>
__global__ __launch_bounds__(64 * MXS_W) __attribute__((amdgpu_waves_per_eu(4))) void mx_stream_kernel(
    const uint8_t *__restrict__ x, const uint8_t *__restrict__ w, const uint8_t *__restrict__ ws, int K, int N, int M, int RT, int wk, int chunk, int inv, void *y,
    int y_bf16, const uint8_t *__restrict__ xs, const int32_t *__restrict__ offsets, int E, bool clear_rest, const int32_t *__restrict__ xrows,
    const uint8_t *__restrict__ w2, const uint8_t *__restrict__ w2s) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr int W = MXS_W, NB = GATED ? 2 : 1, UB = X4 ? 128 : 512, SP = 8 * D + 8;  // bytes of a unit of an activation row; of a row's scales in LDS
    constexpr int SCALES = W * (NB + X4 * MT) * 8 * SP;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, kg = lane >> 4;
    const int kp = wave & ((1 << wk) - 1), G = K >> 5, U = (G + 7) >> 3, rounds = (U + (D << wk) - 1) / (D << wk);
    const int nwg = blockIdx.y * ((W >> wk) * RT), n0 = nwg + (wave >> wk) * RT;
    MxTile t = {0, (int)blockIdx.x * (8 * MT), M - (int)blockIdx.x * (8 * MT), 0, 0};
    if constexpr (GROUPED) {
        t = MxTiles{offsets, E, M, 8 * MT}.find(blockIdx.x);
        if (t.group < 0) {
            if (clear_rest) mx_clear(y, y_bf16, N, t, nwg, (W >> wk) * RT);
            return;
        }
        t = {uniform(t.group), uniform(t.row0), uniform(t.rows), 0, 0};
    }
    const int rows = t.rows < 8 * MT ? t.rows : 8 * MT;

    // ---- activations: rows of a chunk, 16 bytes apart beyond their KiB (eight rows' two halves then cover the banks)
    const int xrow = X4 ? K >> 1 : K * 2, rbytes = (D << wk) * UB, per = (chunk * rbytes + 1023) >> 10, pitch = per * 1024 + 16;
    uint8_t *const xlds = lds + SCALES;
    auto stage = [&](int round) {
        for (int i = wave; i < rows * per; i += W) {  // past a row's end nothing is read and zeros arrive
            const int r = (i * inv) >> 16, b = (i - r * per) * 1024, at = round * rbytes + b + lane * 16;
            const int src = GATED ? __builtin_amdgcn_readfirstlane(xrows[t.row0 + r]) : t.row0 + r;
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(uniform(x + (size_t)src * xrow), 0, xrow, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void *)(xlds + r * pitch + b), 16, at < xrow ? (uint32_t)at : 0x80000000u, 0, 0, 0);
        }
    };
    stage(0);

    // ---- weights: the lane's row and block of a unit
    const int wr = l16 >> 1, wb = (l16 & 1) * 4 + kg;
    const uint8_t *wrow[NB], *srow[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        int n = n0 + (wr < RT ? wr : RT - 1);
        n = n < N ? n : N - 1;
        const size_t r = (size_t)t.group * N + n;
        wrow[i] = (i ? w2 : w) + r * (size_t)(K >> 1);
        srow[i] = (i ? w2s : ws) + r * (size_t)G;
    }
    const int xr = l16 & 7, xb = (l16 >> 3) * 4 + kg;  // the lane's activation row and block
    int xm[MT];
#pragma unroll
    for (int a = 0; a < MT; ++a) xm[a] = a * 8 + xr < rows ? a * 8 + xr : rows - 1;
    u32x4 q[D][NB];
    MxScales<D> s[NB], sx[MT];
    auto first_unit = [&](int round) { return ((round << wk) + kp) * D; };
    auto load_w = [&](int round, int d) {
        int b = (first_unit(round) + d) * 8 + wb;
        b = b < G ? b : G - 1;
#pragma unroll
        for (int i = 0; i < NB; ++i) q[d][i] = load_nt_b128(wrow[i] + (size_t)b * 16);
    };
    auto load_s = [&](int round) {
        const int at = first_unit(round) * 8;
#pragma unroll
        for (int i = 0; i < NB; ++i) s[i].load(srow[i], at + wb * D, G);
        if constexpr (X4)
#pragma unroll
            for (int a = 0; a < MT; ++a) sx[a].load(xs + (size_t)(t.row0 + xm[a]) * G, at + xb * D, G);
    };
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    load_s(0);
#pragma unroll
    for (int d = 0; d < D; ++d) load_w(0, d);
    __builtin_amdgcn_sched_barrier(0);

    f32x4 acc[MT][NB];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[a][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const uint8_t *xl[MT];
#pragma unroll
    for (int a = 0; a < MT; ++a) xl[a] = xlds + xm[a] * pitch + xb * (UB / 8) + kp * D * UB;
    uint8_t *const sl = lds + wave * ((NB + X4 * MT) * 8 * SP);
    wait_vmcnt<NB + X4 * MT + D * NB>();  // what has been requested since the activations
    wg_barrier();
    int at = 0;  // of the round in its chunk
    auto put_scales = [](uint8_t *d, const MxScales<D> &v) { *reinterpret_cast<typename MxScales<D>::bytes_t *>(d) = v.get(); };
    auto turn = [&](int round, bool more) {
        uint32_t sc[NB][D], sxc[MT][D];
#pragma unroll
        for (int i = 0; i < NB; ++i) put_scales(sl + (i * 8 + wr) * SP + wb * D, s[i]);
        if constexpr (X4)
#pragma unroll
            for (int a = 0; a < MT; ++a) put_scales(sl + ((NB + a) * 8 + xr) * SP + xb * D, sx[a]);
        asm volatile("" ::: "memory");  // a wave's LDS accesses keep their order
#pragma unroll
        for (int d = 0; d < D; ++d) {
#pragma unroll
            for (int i = 0; i < NB; ++i) sc[i][d] = sl[(i * 8 + wr) * SP + d * 8 + wb];
            if constexpr (X4)
#pragma unroll
                for (int a = 0; a < MT; ++a) sxc[a][d] = sl[((NB + a) * 8 + xr) * SP + d * 8 + xb];
        }
        asm volatile("" ::: "memory");
        if (more) load_s(round + 1);
        const int left = U - first_unit(round);  // units of the wave in this round
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (more || d < left) {
                const int o = (at * (D << wk) + d) * UB;
                if constexpr (X4) {
#pragma unroll
                    for (int a = 0; a < MT; ++a) {
                        const i32x8 xo = mx_operand(*reinterpret_cast<const u32x4 *>(xl[a] + o));
#pragma unroll
                        for (int i = 0; i < NB; ++i)
                            acc[a][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(q[d][i]), xo, acc[a][i], 4, 4, 0, (int)sc[i][d], 0, (int)sxc[a][d]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        bf16x8 wo[NB];
#pragma unroll
                        for (int i = 0; i < NB; ++i) wo[i] = dequant8_mx(q[d][i][j], mx_scale(sc[i][d]));
#pragma unroll
                        for (int a = 0; a < MT; ++a) {
                            const bf16x8 xo = *reinterpret_cast<const bf16x8 *>(xl[a] + o + j * 16);
#pragma unroll
                            for (int i = 0; i < NB; ++i) acc[a][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wo[i], xo, acc[a][i], 0, 0, 0);
                        }
                    }
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
        if (at == chunk) {
            wg_barrier();
            stage(round + 1);
            wait_vmcnt<0>();
            wg_barrier();
            at = 0;
        }
    }
    turn(round, false);

    // ---- results.  Lane (kg, m < 8): n = 2 kg and 2 kg + 1 of row m; the odd rows' half comes from column 8 + m
    f32x2 out[MT][NB];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int i = 0; i < NB; ++i)
            out[a][i] = f32x2{acc[a][i].x + dpp_f32<0x128, 0xF>(acc[a][i].y), acc[a][i].z + dpp_f32<0x128, 0xF>(acc[a][i].w)};  // row_ror:8
    auto put = [&](int a, int m, int n, f32x2 g, f32x2 u) {
        if (a * 8 + m >= rows) return;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int c = n + e;
            if (2 * kg + e < RT && c < N) store_sum(reinterpret_cast<float *>(y), (size_t)(t.row0 + a * 8 + m) * N + c, GATED ? silu_mul(g[e], u[e]) : g[e], y_bf16);
        }
    };
    if (wk == 0) {
        if (l16 < 8)
#pragma unroll
            for (int a = 0; a < MT; ++a) put(a, l16, n0 + 2 * kg, out[a][0], out[a][NB - 1]);
        return;
    }
    f32x2 *const part = reinterpret_cast<f32x2 *>(xlds);
    wg_barrier();
    if (l16 < 8)
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int i = 0; i < NB; ++i) part[((wave * MT + a) * NB + i) * 32 + kg * 8 + l16] = out[a][i];
    wg_barrier();
    if (kp != 0 || l16 >= 8) return;
#pragma unroll
    for (int a = 0; a < MT; ++a) {
        f32x2 v[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            v[i] = out[a][i];
            for (int k = 1; k < 1 << wk; ++k) v[i] += part[(((wave + k) * MT + a) * NB + i) * 32 + kg * 8 + l16];
        }
        put(a, l16, n0 + 2 * kg, v[0], v[NB - 1]);
    }
}

// Weight rows of a wave, and how many waves split K (log2): as many rows to a workgroup as give every compute unit the same number of them; waves that
// they leave split K
struct StreamShape {
    int RT, wk;
    int64_t cols(int N) const { return mx_ceil(N, (MXS_W >> wk) * RT); }  // workgroups along n
};
static StreamShape stream_shape(const MxProduct &p) {
    if (p.offsets) return {8, 0};
    const int64_t turns = mx_ceil(p.N, 256 * 64);
    const int rows = (int)mx_ceil(p.N, 256 * turns), wk = rows > 32 ? 0 : rows > 16 ? 1 : rows > 8 ? 2 : 3, s = MXS_W >> wk;
    return {(rows + s - 1) / s, wk};
}

template <bool X4, bool GATED, bool GROUPED, int MT, int D>
static int launch(const MxProduct &p, StreamShape shape, hipStream_t st) {
    constexpr int W = MXS_W, NB = GATED ? 2 : 1, UB = X4 ? 128 : 512, SCALES = W * (NB + X4 * MT) * 8 * (8 * D + 8);
    const int RT = shape.RT, wk = shape.wk;
    const int U = (p.K + 255) / 256, round = D << wk, rounds = (U + round - 1) / round, rows = p.M < 8 * MT ? p.M : 8 * MT;
    const int64_t tiles = p.offsets ? mx_most_tiles(p.M, p.E, 8 * MT) : mx_ceil(p.M, 8 * MT), cols = shape.cols(p.N);
    if (tiles > (1 << 22) || cols > kStreamCols) return fail(CHADQ_ERR_SHAPE, "mxfp4 product: M=%d N=%d are too many tiles", p.M, p.N);
    // all of K if it fits: two workgroups to a compute unit where there are so many
    const int most = (tiles * cols <= 256 ? 147456 : 73728) / (rows * round * UB), chunk = most < 1 ? 1 : most > rounds ? rounds : most;
    const size_t per = ((size_t)chunk * round * UB + 1023) / 1024, xb = rows * (per * 1024 + 16), part = wk ? W * MT * NB * 256 : 0;
    const size_t lds = SCALES + (part > xb ? part : xb);
    if (lds > 163840) return fail(CHADQ_ERR_SHAPE, "mxfp4 product: %zu bytes of LDS", lds);
    const auto kernel = &mx_stream_kernel<X4, GATED, GROUPED, MT, D>;
    static std::atomic<bool> set[64];  // more LDS than the default limit: once per device
    int dev = 0;
    CHADQ_HIP(hipGetDevice(&dev));
    if (dev >= 64 || !set[dev].load()) {
        CHADQ_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 163840));
        if (dev < 64) set[dev].store(true);
    }
    hipLaunchKernelGGL(kernel, dim3((int)tiles, (int)cols), dim3(64 * W), lds, st, reinterpret_cast<const uint8_t *>(p.x), p.w, p.ws, p.K, p.N, p.M, RT, wk, chunk,
                       65536 / (int)per + 1, p.y, (int)p.y_bf16, p.xs, p.offsets, p.E, p.clear_rest, p.rows, p.w2, p.w2s);
    return hip_check(hipGetLastError(), "mxfp4 product launch");
}

template <bool X4, bool GATED, bool GROUPED, int MT>
static int launch_rows(const MxProduct &p, hipStream_t st) {
    const int U = (p.K + 255) / 256;
    const StreamShape shape = stream_shape(p);
    if constexpr (GROUPED) {
        return U > 2 ? launch<X4, GATED, true, MT, 4>(p, shape, st) : launch<X4, GATED, true, MT, 1>(p, shape, st);
    } else {
        const int wk = shape.wk, own = (U + (1 << wk) - 1) >> wk;
        const int fit = 131072 / ((p.M < 16 ? p.M : 16) * (X4 ? 128 : 512) << wk), most = own < fit ? own : fit;
        // (MXFP4 x: eight registers for an operand that uses four, so eight units ahead would not fit)
        if constexpr (!X4)
            if (most > 4) return launch<X4, GATED, GROUPED, MT, 8>(p, shape, st);
        return most > 2   ? launch<X4, GATED, GROUPED, MT, 4>(p, shape, st)
               : most > 1 ? launch<X4, GATED, GROUPED, MT, 2>(p, shape, st)
                          : launch<X4, GATED, GROUPED, MT, 1>(p, shape, st);
    }
}

int mx_stream_launch(const MxProduct &p, hipStream_t st) {
    if (p.w2) return launch_rows<false, true, true, 1>(p, st);
    if (p.offsets) return p.xs ? launch_rows<true, false, true, 1>(p, st) : launch_rows<false, false, true, 1>(p, st);
    if (p.M <= 8) return p.xs ? launch_rows<true, false, false, 1>(p, st) : launch_rows<false, false, false, 1>(p, st);
    return p.xs ? launch_rows<true, false, false, 2>(p, st) : launch_rows<false, false, false, 2>(p, st);
}

// Up to 16 rows, or 8 of a group on average, stream the weights, more go through the tiles.  By group, 8 matrices of 14336 x 4096, us, streamed / tiles, bf16 x: 40
// rows evenly 45 / 59, 64 evenly 48 / 59, 72 evenly 81 / 60 (a group of more than eight rows reads its weights again).  Of the groups the rule knows the mean alone:
// drawn at random 40 rows take 53 / 59, 56 rows 63 / 59, 64 rows 64 / 57, 80 rows 79 / 60; all in one group 40 rows 34 / 26, 64 rows 49 / 26.  MXFP4 x, 16 matrices of
// 4096 x 2048, 64 of 1024 x 2048 and 4 of 4096 x 4096 cross between 6 and 8 rows a group too.
// Columns beyond what the streaming grid holds (4194240) go through the tiles whatever the rows.
bool mx_streams(const MxProduct &p) { return (p.offsets ? p.M <= (int64_t)8 * p.E : p.M <= 16) && stream_shape(p).cols(p.N) <= kStreamCols; }

int mx_product_part_k(const MxProduct &p, int most_parts) { return mx_streams(p) || !mx_tile_ok(p) ? 0 : mx_tile_pick(p, most_parts).part_k; }

size_t mx_product_workspace_bytes(int M, int N, int K, bool x_mxfp4) {
    MxProduct p = {};
    p.M = M;
    p.N = N;
    p.K = K;
    p.E = 1;
    static const uint8_t any = 0;
    p.xs = x_mxfp4 ? &any : nullptr;
    p.part_k = mx_product_part_k(p, kMxParts);
    return p.part_k ? (size_t)p.parts() * M * N * 4 : 0;
}

int mx_product_launch(const MxProduct &p, void *workspace, size_t workspace_bytes, hipStream_t st) {
    if (mx_streams(p) || !mx_tile_ok(p)) return mx_stream_launch(p, st);
    if (p.part_k) return mx_tile_launch(p, mx_tile_pick(p, kMxGroupParts).tile, st);  // (the caller, who asked for at most so many, joins the parts)
    if (!p.offsets && workspace) {
        MxProduct q = p;
        const MxTilePick pick = mx_tile_pick(p, kMxParts);
        q.part_k = pick.part_k;
        if (pick.part_k && workspace_bytes >= (size_t)q.parts() * p.M * p.N * 4) return mx_tile_parts_launch(q, pick.tile, reinterpret_cast<float *>(workspace), st);
    }
    return mx_tile_launch(p, mx_tile_pick(p, 1).tile, st);
}

}  // namespace chadq
