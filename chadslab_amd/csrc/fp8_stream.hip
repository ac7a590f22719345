// Products of at most 16 rows (of a group) on FP8 weights, x bf16 or FP8, one matrix or one per group of rows.  HBM-bound: every weight is read once per tile of 8 MT rows.
//
// A wave works on 8 weight rows and one block of 128 k at a time (a unit): one load instruction brings 128 consecutive bytes of each row, 16 to a lane, straight into
// the registers.  They become bf16, exactly, one conversion per pair, and so do 8-bit activations: v_mfma_f32_16x16x32_bf16 sums exact products in fp32, where the
// 8-bit matrix instructions add eight products as multiples of 2^-13 of the largest and lose what lies below.  That instruction has 16 weight rows and 4 pieces of
// k; so each row takes two of its rows, with one half of its eight pieces each, and the activations take two columns each, row m's halves in column m and in column
// 8 + m: of the result the (even row, column m) and (odd row, column 8 + m) are added and multiplied with the block's scales.  MT = 2: rows 8-15 by
// a second pair of instructions.
// A workgroup's eight waves are S = 8 / WK side by side in n and WK along K.  A round is D units of each wave; its weights are requested a round ahead.  The activations
// and all scales wait in LDS, a chunk of rounds at a time, requested before the first weights; behind K the activations are zeros, and a lane past the end of its weight
// row reads that row's last bytes again.
// us: 1 x 14336 x 4096 10.6 (the weights in turn with others: 5.5 TB/s), 6 x 11008 x 4096 with 8-bit x 9.5, 32 rows by group on 8 of 14336 x 4096 73 (470 MB, 6.4 TB/s, some from the
// last-level cache).  The first form, a row's weights by one lane each, took 35.7, 36.5 and 223.
#include "fp8.h"

namespace chadq {

constexpr int F8S_W = 8;  // waves
constexpr int kFp8StreamCols = 65535;  // workgroups along n: a grid's second dimension

// 16 or 4 bytes a lane from a row of `bytes`, the lane's from `at` on, one behind the other to dst; zeros behind the row's end
__device__ __forceinline__ void to_lds16(const void *row, int bytes, uint8_t *dst, int at) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(uniform(row), 0, bytes, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void *)dst, 16, at < bytes ? (uint32_t)at : 0x80000000u, 0, 0, 0);
}
__device__ __forceinline__ void to_lds4(const void *row, int bytes, uint8_t *dst, int at) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(uniform(row), 0, bytes, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void *)dst, 4, at < bytes ? (uint32_t)at : 0x80000000u, 0, 0, 0);
}

// What the first requests need comes first in the arguments, where it arrives in registers with the wave.
// RT: weight rows of a wave in use (<= 8); wk: log2 WK; chunk: rounds of a chunk; inv: 65536 / KiB of its activation rows, rounded up
// GATED: gate rows w and up rows w2, silu(gate) up
template <bool X8, bool GATED, bool GROUPED, int MT, int D>
__global__ __launch_bounds__(64 * F8S_W) __attribute__((amdgpu_waves_per_eu(4))) void fp8_stream_kernel(
    const uint8_t *__restrict__ x, const uint8_t *__restrict__ w, const float *__restrict__ ws, int K, int N, int M, int RT, int wk, int chunk, int inv, void *y,
    int y_bf16, const float *__restrict__ xs, const int32_t *__restrict__ offsets, int E, bool clear_rest, const int32_t *__restrict__ xrows,
    const uint8_t *__restrict__ w2, const float *__restrict__ w2s) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    constexpr int W = F8S_W, NB = GATED ? 2 : 1, UB = X8 ? 128 : 256, PAD = X8 ? 32 : 16;  // UB: bytes of a unit of an activation row
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, kg = lane >> 4;
    const int kp = wave & ((1 << wk) - 1), U = (K + 127) >> 7, rounds = (U + (D << wk) - 1) / (D << wk);
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

    // ---- requests into LDS, past the end of a row nothing is read and zeros arrive.  Scales: those of the two blocks of rows that the workgroup's (at most 64)
    // weight rows lie in, and of each activation row, S floats apart; then the activation rows, PAD bytes apart beyond their KiB (the 16 lanes that read
    // at a time then cover the banks)
    const int units = chunk * (D << wk), sq = (units + 63) >> 6, S = sq * 64 + 1;
    const int xrow = X8 ? K : K * 2, rbytes = units * UB, per = (rbytes + 1023) >> 10, pitch = per * 1024 + PAD;
    uint8_t *const xlds = lds + (((NB * 2 + (X8 ? rows : 0)) * S * 4 + 15) & ~15);
    const int GN = (N + 127) >> 7, nb0 = nwg >> 7;
    auto source = [&](int r) { return GATED ? __builtin_amdgcn_readfirstlane(xrows[t.row0 + r]) : t.row0 + r; };
    auto stage = [&](int round) {
        const int u0 = round * (D << wk);
        for (int i = wave; i < rows * per; i += W) {
            const int r = (i * inv) >> 16, b = (i - r * per) * 1024;
            to_lds16(x + (size_t)source(r) * xrow, xrow, xlds + r * pitch + b, u0 * UB + b + lane * 16);
        }
        for (int i = wave; i < NB * 2 + (X8 ? rows : 0); i += W) {
            const int nb = nb0 + (i & 1) < GN ? nb0 + (i & 1) : GN - 1;
            const float *const row = i < NB * 2 ? (i >> 1 ? w2s : ws) + ((size_t)t.group * GN + nb) * U : xs + (size_t)source(i - NB * 2) * U;
            for (int c = 0; c < sq; ++c) to_lds4(row, U * 4, lds + (i * S + c * 64) * 4, (u0 + c * 64 + lane) * 4);
        }
    };
    // Workgroups that all go through k alike meet in a few of the memory's channels where rows are a large power of two apart: each begins at a chunk and a round in it of its own and
    // goes round (where the last one is whole).  us, all from 0 / each from its own, weights from memory: 1 x 14336 x 4096 11.8 / 10.6, 8 x 8192 x 8192 17.8 / 13.0, 16 x 4096 x 4096
    // 7.4 / 6.8, 64 rows by group on 32 of 4096 x 8192 199 / 156; with rows of 2048, 7168 and 14336 bytes alike
    const int own = U % (D << wk) == 0 ? (int)blockIdx.y + 3 * t.group : 0;
    int len = rounds < chunk ? rounds : chunk;  // the chunk's rounds
    const int start = GROUPED && len < rounds && rounds % len == 0 ? own / len * len % rounds : 0;
    int base = start;  // the first of them
    stage(base);
    const int first = own % len;
    int at = first;  // the round in it

    // ---- weights: the lane's row and piece of a unit
    const int wr = l16 >> 1, wb = X8 ? kg * 2 + (l16 & 1) : (l16 & 1) * 4 + kg, pieces = K >> 4;
    const uint8_t *wrow[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        int n = n0 + (wr < RT ? wr : RT - 1);
        n = n < N ? n : N - 1;
        wrow[i] = (i ? w2 : w) + ((size_t)t.group * N + n) * (size_t)K;
    }
    const int xr = l16 & 7, xb = X8 ? kg * 2 + (l16 >> 3) : (l16 >> 3) * 4 + kg;  // the lane's activation row and piece
    u32x4 q[D][NB];
    auto first_unit = [&](int round) { return ((round << wk) + kp) * D; };
    auto load_w = [&](int round, int d) {
        int b = (first_unit(round) + d) * 8 + wb;
        b = b < pieces ? b : pieces - 1;
#pragma unroll
        for (int i = 0; i < NB; ++i) q[d][i] = load_nt_b128(wrow[i] + (size_t)b * 16);
    };
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < D; ++d) load_w(base + at, d);
    __builtin_amdgcn_sched_barrier(0);

    // the sums of lane (kg, m < 8): weight rows 2 kg and 2 kg + 1, activation row m
    f32x2 acc[MT][NB];
#pragma unroll
    for (int a = 0; a < MT; ++a)
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[a][i] = f32x2{0.f, 0.f};
    const uint8_t *xl[MT];
    const float *sxl[MT], *swl[2];
#pragma unroll
    for (int a = 0; a < MT; ++a) {
        const int xm = a * 8 + xr < rows ? a * 8 + xr : rows - 1;
        xl[a] = xlds + xm * pitch + xb * (UB / 8) + kp * D * UB;
        sxl[a] = reinterpret_cast<const float *>(lds) + (NB * 2 + xm) * S + kp * D;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        int n = n0 + 2 * kg + e;
        n = n < N ? n : N - 1;
        const int b = (n >> 7) - nb0;
        swl[e] = reinterpret_cast<const float *>(lds) + (b < 1 ? b : 1) * S + kp * D;  // (rows of no use to anyone may lie further)
    }
    wait_vmcnt<D * NB>();  // what has been requested since the activations
    wg_barrier();
    auto turn = [&](int next, bool more) {
        const int left = U - first_unit(base + at);  // units of the wave in this round
#pragma unroll
        for (int d = 0; d < D; ++d) {
            if (more || d < left) {
                const int u = at * (D << wk) + d, o = u * UB;
                bf16x8 wo[NB][2];
#pragma unroll
                for (int i = 0; i < NB; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const u32x2 lo = fp8_to_bf16(q[d][i][2 * j]), hi = fp8_to_bf16(q[d][i][2 * j + 1]);
                        wo[i][j] = __builtin_bit_cast(bf16x8, u32x4{lo.x, lo.y, hi.x, hi.y});
                    }
#pragma unroll
                for (int a = 0; a < MT; ++a) {
                    bf16x8 xo[2];
                    if constexpr (X8) {
                        const u32x4 v = *reinterpret_cast<const u32x4 *>(xl[a] + o);
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const u32x2 lo = fp8_to_bf16(v[2 * j]), hi = fp8_to_bf16(v[2 * j + 1]);
                            xo[j] = __builtin_bit_cast(bf16x8, u32x4{lo.x, lo.y, hi.x, hi.y});
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 2; ++j) xo[j] = *reinterpret_cast<const bf16x8 *>(xl[a] + o + j * 16);
                    }
#pragma unroll
                    for (int i = 0; i < NB; ++i) {
                        f32x4 r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int j = 0; j < 2; ++j) r = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wo[i][j], xo[j], r, 0, 0, 0);
                        f32x2 s = {swl[0][i * 2 * S + u], swl[1][i * 2 * S + u]};
                        if constexpr (X8) s *= sxl[a][u];
                        // (the halves before the scales: one half's sum may be 0 beside an infinite scale; row_ror:8)
                        acc[a][i].x = __builtin_fmaf(r.x + dpp_f32<0x128, 0xF>(r.y), s.x, acc[a][i].x);
                        acc[a][i].y = __builtin_fmaf(r.z + dpp_f32<0x128, 0xF>(r.w), s.y, acc[a][i].y);
                    }
                }
            }
            if (more) load_w(next, d);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (;;) {
        for (int i = 1; i < len; ++i) {
            const int next = at + 1 == len ? 0 : at + 1;
            turn(base + next, true);
            at = next;
        }
        const int begin = base + len == rounds ? 0 : base + len;
        if (begin == start) break;
        const int size = rounds - begin < chunk ? rounds - begin : chunk, next = first < size ? first : 0;
        turn(begin + next, true);
        base = begin;
        len = size;
        at = next;
        wg_barrier();
        stage(base);
        wait_vmcnt<0>();
        wg_barrier();
    }
    turn(0, false);

    // ---- results.  Lane (kg, m < 8): n = 2 kg and 2 kg + 1 of row m
    auto put = [&](int a, f32x2 g, f32x2 u) {
        if (a * 8 + l16 >= rows) return;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int c = n0 + 2 * kg + e;
            if (2 * kg + e < RT && c < N) store_sum(reinterpret_cast<float *>(y), (size_t)(t.row0 + a * 8 + l16) * N + c, GATED ? silu_mul(g[e], u[e]) : g[e], y_bf16);
        }
    };
    if (wk == 0) {
        if (l16 < 8)
#pragma unroll
            for (int a = 0; a < MT; ++a) put(a, acc[a][0], acc[a][NB - 1]);
        return;
    }
    f32x2 *const part = reinterpret_cast<f32x2 *>(xlds);
    wg_barrier();
    if (l16 < 8)
#pragma unroll
        for (int a = 0; a < MT; ++a)
#pragma unroll
            for (int i = 0; i < NB; ++i) part[((wave * MT + a) * NB + i) * 32 + kg * 8 + l16] = acc[a][i];
    wg_barrier();
    if (kp != 0 || l16 >= 8) return;
#pragma unroll
    for (int a = 0; a < MT; ++a) {
        f32x2 v[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            v[i] = acc[a][i];
            for (int k = 1; k < 1 << wk; ++k) v[i] += part[(((wave + k) * MT + a) * NB + i) * 32 + kg * 8 + l16];
        }
        put(a, v[0], v[NB - 1]);
    }
}

// Weight rows of a wave, and how many waves split K (log2): as many rows to a workgroup as give every compute unit the same number of them; waves that
// they leave split K
struct Fp8StreamShape {
    int RT, wk;
    int64_t cols(int N) const { return mx_ceil(N, (F8S_W >> wk) * RT); }  // workgroups along n
};
static Fp8StreamShape stream_shape(const Fp8Product &p) {
    if (p.offsets) return {8, 0};
    const int64_t turns = mx_ceil(p.N, 256 * 64);
    const int rows = (int)mx_ceil(p.N, 256 * turns), wk = rows > 32 ? 0 : rows > 16 ? 1 : rows > 8 ? 2 : 3, s = F8S_W >> wk;
    return {(rows + s - 1) / s, wk};
}

template <bool X8, bool GATED, bool GROUPED, int MT, int D>
static int launch(const Fp8Product &p, Fp8StreamShape shape, hipStream_t st) {
    constexpr int W = F8S_W, NB = GATED ? 2 : 1, UB = X8 ? 128 : 256;
    const int RT = shape.RT, wk = shape.wk;
    const int U = fp8_blocks(p.K), round = D << wk, rounds = (U + round - 1) / round, rows = p.M < 8 * MT ? p.M : 8 * MT;
    const int64_t tiles = p.offsets ? mx_most_tiles(p.M, p.E, 8 * MT) : mx_ceil(p.M, 8 * MT), cols = shape.cols(p.N);
    if (tiles > (1 << 22) || cols > kFp8StreamCols) return fail(CHADQ_ERR_SHAPE, "fp8 product: M=%d N=%d are too many tiles", p.M, p.N);
    // all of K if it fits: two workgroups to a compute unit where there are so many
    const int most = (tiles * cols <= 256 ? 139264 : 69632) / (rows * round * (UB + 4)), chunk = most < 1 ? 1 : most > rounds ? rounds : most;
    const size_t units = (size_t)chunk * round, per = (units * UB + 1023) / 1024, xb = rows * (per * 1024 + (X8 ? 32 : 16)), part = wk ? W * MT * NB * 256 : 0;
    const size_t scales = ((NB * 2 + (X8 ? rows : 0)) * ((units + 63) / 64 * 64 + 1) * 4 + 15) & ~(size_t)15;
    const size_t lds = scales + (part > xb ? part : xb);
    if (lds > 163840) return fail(CHADQ_ERR_SHAPE, "fp8 product: %zu bytes of LDS", lds);
    const auto kernel = &fp8_stream_kernel<X8, GATED, GROUPED, MT, D>;
    static std::atomic<bool> set[64];  // more LDS than the default limit: once per device
    int dev = 0;
    CHADQ_HIP(hipGetDevice(&dev));
    if (dev >= 64 || !set[dev].load()) {
        CHADQ_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, 163840));
        if (dev < 64) set[dev].store(true);
    }
    hipLaunchKernelGGL(kernel, dim3((int)tiles, (int)cols), dim3(64 * W), lds, st, reinterpret_cast<const uint8_t *>(p.x), p.w, p.ws, p.K, p.N, p.M, RT, wk, chunk,
                       65536 / (int)per + 1, p.y, (int)p.y_bf16, p.xs, p.offsets, p.E, p.clear_rest, p.rows, p.w2, p.w2s);
    return hip_check(hipGetLastError(), "fp8 product launch");
}

template <bool X8, bool GATED, bool GROUPED, int MT>
static int launch_rows(const Fp8Product &p, hipStream_t st) {
    const int U = fp8_blocks(p.K);
    const Fp8StreamShape shape = stream_shape(p);
    if constexpr (GROUPED) {
        return U > 4 ? launch<X8, GATED, true, MT, 4>(p, shape, st) : launch<X8, GATED, true, MT, 1>(p, shape, st);
    } else {
        const int wk = shape.wk, own = (U + (1 << wk) - 1) >> wk;  // units of a wave
        if constexpr (MT == 1)  // (more registers than there are for two sets of rows)
            if (own > 4) return launch<X8, GATED, GROUPED, MT, 8>(p, shape, st);
        return own > 2 ? launch<X8, GATED, GROUPED, MT, 4>(p, shape, st)
               : own > 1 ? launch<X8, GATED, GROUPED, MT, 2>(p, shape, st)
                         : launch<X8, GATED, GROUPED, MT, 1>(p, shape, st);
    }
}

int fp8_stream_launch(const Fp8Product &p, hipStream_t st) {
    if (p.w2) return p.xs ? launch_rows<true, true, true, 1>(p, st) : launch_rows<false, true, true, 1>(p, st);
    if (p.offsets) return p.xs ? launch_rows<true, false, true, 1>(p, st) : launch_rows<false, false, true, 1>(p, st);
    if (p.M <= 8) return p.xs ? launch_rows<true, false, false, 1>(p, st) : launch_rows<false, false, false, 1>(p, st);
    return p.xs ? launch_rows<true, false, false, 2>(p, st) : launch_rows<false, false, false, 2>(p, st);
}

// Up to 16 rows, or 8 of a group on average, stream the weights, more go through the tiles.  By group, us streamed / in tiles, bf16 x: 8 of 14336 x 4096, 4 rows to each 73 / 90, 8 to each
// 75 / 92, 12 to each 141 / 92; 64 of 1408 x 2048, the same, 31 / 44, 33 / 44, 61 / 45.  The host does not know how the rows are spread: drawn groups of 8 on average, whose larger ones read
// their weights twice, lose by it (114 / 89, 44 / 43), and so do 4 on average only at many small groups (256 of 1024 x 1024, 58 / 51); all rows in one group, 8 times as many as there
// are groups, 75 / 41.  8-bit x: streamed the same, in tiles up to 12 % less than bf16 (one group
// 40 %; 256 groups 9 % more).
// Columns beyond what the streaming grid holds (4194240) go through the tiles whatever the rows.
bool fp8_streams(const Fp8Product &p) { return (p.offsets ? p.M <= (int64_t)8 * p.E : p.M <= 16) && stream_shape(p).cols(p.N) <= kFp8StreamCols; }

}  // namespace chadq
