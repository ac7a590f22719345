// Products of many rows on FP8 weights, x bf16 or FP8, one matrix or one per group of rows.
//
// A workgroup's WN x WM waves share a tile of TN weight rows x TM activation rows; a wave sums NB x MB blocks of 32 x 32.  The weights are the
// matrix cores' first operand, so that a lane holds four consecutive n of one activation row.
//   FP8 x   v_mfma_f32_16x16x128_f8f6f4 takes a whole scale block of k: its result, from 0, times the block's two scales is added to the sum by FMAs that
//           follow some instructions behind.  The instruction adds eight products as multiples of 2^-13 of the largest: 2^-16 of a result's norm on normal data, beside
//           the up to 2^-8 of its rounding to bf16.  (32x32x64, two to a block: 3.3 instead of 3.6 PFLOP/s with the FMAs, from registers)
//   bf16 x  the values become bf16, exactly, v_mfma_f32_32x32x16_bf16; the sums of a block begin from 0 and are added, times its scale, when the next begins
// A step is SK of K.  Values and activations go global -> LDS by DMA, ST stages, requests dealt to the waves in equal numbers and placed between
// the MFMAs; a piece past the end of a row or of the matrix is requested beyond the buffer's range and arrives as zeros, so nothing in the loop knows about
// edges.  Scales: a thread loads two steps' of a row of x, or of a block of weight rows, two steps ahead, and puts them into LDS.  16-byte
// pieces of a row are XOR-swizzled by the row so that the 16 rows that a read takes at a time cover all banks.  WK > 1: waves of a workgroup split the k of a
// step and add their sums at the end, so that a small tile too has eight waves to hide its reads.
// us, matrix cores' busy share: 4096 x 14336 x 4096 8-bit 234-241, 51 % (2.0 PFLOP/s; 256 x 256); 1000 x 4096 x 14336 bf16 124-130, 47 % (0.9 PFLOP/s; 128 x 128, one round); 2048 rows by group on
// 16 of 4096 x 2048 8-bit 42-46, 22 %; gate and up of 6000 pairs, 64 experts of 1408 x 2048, 111, 19 % (407 MB, 3.7 TB/s).  Of 4096^3 with 256 x 256 tiles, 69 us, some 8 are outside
// the loop, 13 are the requests and 9 the scales' FMAs; the MFMAs alone take 32.
#include <cmath>
#include <type_traits>
#include <utility>

#include "fp8.h"

namespace chadq {
namespace f8t {

template <bool X8_, bool GATED_, int WN_, int WM_, int WK_, int NB_, int MB_, int SK_, int ST_>
struct Cfg {
    static constexpr bool X8 = X8_, GATED = GATED_;
    static constexpr int WN = WN_, WM = WM_, WK = WK_, NB = NB_, MB = MB_, SK = SK_, ST = ST_;
    static constexpr int NW = WN * WM * WK, T = 64 * NW, TN = 32 * NB * WN, TM = 32 * MB * WM, TO = GATED ? TN / 2 : TN;  // TO: result columns
    // a weight row's bytes per step in parts of WROW, one for each wave along K, and an activation row's in parts of 128.  FP8 x: a part is a block; bf16: half a
    // block, the other half comes with the next step, so that a wave sums whole blocks
    static constexpr int WROW = X8 ? 128 : 64, WPARTS = SK / WROW, XPARTS = WPARTS;
    static constexpr int W_STAGE = TN * SK, X_STAGE = TM * 128 * XPARTS;
    // DMA instructions per wave and step, as many for each (what is too many of them for few rows fills a place nobody reads)
    static constexpr int WI = W_STAGE / (1024 * NW), XI = (X_STAGE + 1024 * NW - 1) / (1024 * NW), REQ = WI + XI, STAGE = W_STAGE + XI * 1024 * NW;
    static_assert(WI * 1024 * NW == W_STAGE && X_STAGE % 1024 == 0, "whole DMA instructions");
    // of a step's requests so many come before position pos of its NP: with two stages they are waited for at the end of the same step, so they come in its first half
    static constexpr int requested(int pos, int np) { return ST > 2 ? pos * REQ / np : 2 * pos < np ? 2 * pos * REQ / np : REQ; }
    static constexpr int GE = 2 * SK / 128;                                      // scales of a row in two steps, loaded together (a group)
    static constexpr int SROWS = (X8 ? TM : 0) + 2, SPITCH = (SROWS + 31) / 32 * 32;  // rows of scales: of x, of the tile's two blocks of weight rows (gate and up)
    static_assert(SROWS <= T && WPARTS == WK, "a thread to a row of scales; each wave a part");
    static constexpr int S_OFF = ST * STAGE, S_GROUP = GE * SPITCH * 4, DUMP = S_OFF + 2 * S_GROUP, OPER = DUMP + 64 * GE * 4, RED = WN * WM * (WK - 1) * NB * MB * 4096;
    static constexpr bool H8 = X8 && GATED && TO == 128;  // results in 8 bits: a tile has whole blocks of them
    static constexpr int EPI = TM * (TO * (H8 ? 4 : 2) + 16), MOST = OPER > RED ? OPER : RED, LDS = MOST > EPI ? MOST : EPI;
    static_assert(LDS <= 163840, "LDS of a compute unit");
    static_assert(!GATED || (NB % 2 == 0 && 1024 / WROW <= 32), "gate and up blocks side by side; a DMA instruction's rows are of one block");
};

// f(0), f(1), ... with the numbers as types
template <typename F, int... S>
__device__ __forceinline__ void each(F &f, std::integer_sequence<int, S...>) {
    (f(std::integral_constant<int, S>{}), ...);
}

// how the 16-byte pieces of row r are permuted: rows of 64 bytes, four of them to the banks, or of 128, two
template <int ROW>
__device__ __forceinline__ int key(int r) {
    return ROW == 64 ? (r >> 2) & 3 : (r >> 1) & 7;
}

__device__ const float kNoScales[16] = {};

// What a workgroup reads: its requests, its scales
template <typename C>
struct Source {
    const Fp8Product &p;
    uint8_t *const lds;
    int tid = 0, lane = 0, wave = 0, s0 = 0, kend = 0, steps = 0, nrows = 0;  // s0: first step of the workgroup's part of K; nrows: result columns that there are
    int groups = 1, turn = 0;  // of two steps; which of them is the first
    __amdgpu_buffer_rsrc_t wrsrc, w2rsrc, xrsrc;
    // of the lane's piece in a part of a row (the rows of a wave's requests of a kind are a multiple of 16 apart), and in a request's rows
    int wplace = 0, xplace = 0;
    uint32_t wlane = 0, xlane[C::GATED ? C::XI : 1];  // (GATED: rows through an index, each from x's first)
    int wbytes = 0, xbytes = 0;  // of a row
    const __attribute__((address_space(1))) float *srow = nullptr;
    int whole = 0;
    float sv[C::GE], tail[C::GE];
    static constexpr uint32_t kOut = 0x80000000u;

    __device__ __forceinline__ Source(const Fp8Product &p, const MxTile &t, int n0, uint8_t *lds) : p(p), lds(lds) {
        tid = threadIdx.x;
        lane = tid & 63;
        wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        s0 = p.part_k ? (int)blockIdx.y * (p.part_k / C::SK) : 0;
        kend = p.part_k && s0 * C::SK + p.part_k < p.K ? s0 * C::SK + p.part_k : p.K;
        steps = (kend - s0 * C::SK + C::SK - 1) / C::SK;
        nrows = p.N - n0 < C::TO ? p.N - n0 : C::TO;
        groups = (steps + 1) / 2;
        // Groups' weights come from memory once, and rows a large power of two apart (or a multiple of it) share its channels: workgroups that all go through k alike meet in a
        // few of them.  So by group each begins at a k of its own and goes round.  us, all from 0 / each from its own, 24 rows a group: 32 of 4096 x 4096 8-bit 130 / 94, bf16 138 / 99; 8 of
        // 8192 x 8192 116 / 102 and 127 / 97; 94 rows on average, 32 of 4096 x 4096 149 / 129 and 203 / 199.  Rows of 1408, 1536 and 2560 bytes, which lie in all channels anyhow: 8-bit alike
        // within 2 %, bf16 2 to 3 % behind a form that knows no turn, and as much if these alone began at 0: it is the arithmetic, not the order, so there is no rule by length.  One
        // matrix for all rows gains up to 8 % (28672 x 8192, 20 rows) or loses 25 % (48 rows) and stays as it is.
        turn = p.offsets ? (n0 / C::TO + 3 * t.group) % groups : 0;
        wbytes = p.K;
        xbytes = C::X8 ? p.K : p.K * 2;
        const size_t wfirst = (size_t)t.group * p.N + n0;
        wrsrc = __builtin_amdgcn_make_buffer_rsrc(uniform(p.w + wfirst * wbytes), 0, uniform(nrows * wbytes), 0x00020000);
        w2rsrc = C::GATED ? __builtin_amdgcn_make_buffer_rsrc(uniform(p.w2 + wfirst * wbytes), 0, uniform(nrows * wbytes), 0x00020000) : wrsrc;
        xrsrc = __builtin_amdgcn_make_buffer_rsrc(uniform(reinterpret_cast<const uint8_t *>(p.x) + (C::GATED ? (size_t)0 : (size_t)t.row0 * xbytes)), 0,
                                                  uniform((C::GATED ? p.x_rows : t.rows) * xbytes), 0x00020000);
        static_assert(C::NW * 64 / (C::WROW / 16) % 16 == 0 && C::NW * 8 % 16 == 0, "rows of a wave's requests");
        constexpr int PPR = C::WROW / 16;  // pieces of a row of weights
        wplace = 16 * ((lane % PPR) ^ key<C::WROW>(wave * (64 / PPR) + lane / PPR));
        xplace = 16 * ((lane % 8) ^ key<128>(wave * 8 + lane / 8));
        wlane = (uint32_t)(lane / PPR) * (uint32_t)wbytes + wplace;
    }
    // The rest, of which an index may have to be waited for
    __device__ __forceinline__ void rows(const MxTile &t, int n0) {
        if constexpr (C::GATED) {
#pragma unroll
            for (int q = 0; q < C::XI; ++q) {
                const int e = (q * C::NW + wave) * 8 + lane / 8, r = e % C::TM;
                xlane[q] = r < t.rows && e < C::TM * C::XPARTS ? (uint32_t)p.rows[t.row0 + r] * (uint32_t)xbytes + xplace : kOut;
            }
        } else {
            xlane[0] = (uint32_t)(lane / 8) * (uint32_t)xbytes + xplace;
        }
        // scales.  Those of the last group, if it is no whole one, are loaded one by one before the loop (zeros behind the end of the row, where the activations
        // are zeros too).  No branch: a thread without a row loads another one's and writes where nobody reads, and so does the loop behind the last whole group.
        const int G = fp8_blocks(p.K), GN = fp8_blocks(p.N), r = tid < C::SROWS ? tid : 0;
        auto global = [](const float *p) { return (const __attribute__((address_space(1))) float *)p; };
        if (C::X8 && r < C::TM) {
            const int m = t.row0 + (r < t.rows ? r : t.rows - 1);
            srow = global(p.xs) + (size_t)(C::GATED ? p.rows[m] : m) * G;
        } else {
            const int j = r - (C::X8 ? C::TM : 0), nb = (n0 >> 7) + (C::GATED ? 0 : j);
            srow = global(C::GATED && j ? p.w2s : p.ws) + ((size_t)t.group * GN + (nb < GN ? nb : GN - 1)) * G;
        }
        whole = G / C::GE;
#pragma unroll
        for (int e = 0; e < C::GE; ++e) tail[e] = 0.f;
        if (G % C::GE)
#pragma unroll
            for (int e = 0; e < C::GE; ++e)
                if (whole * C::GE + e < G) tail[e] = srow[whole * C::GE + e];
        if (whole == 0) srow = global(kNoScales);  // (readable, for the loop)
    }
    // What comes before the first step: stages 0 .. ST - 2, the weights of the first two in front of everything that waits for an index; ends with stage 0 and the first
    // group's scales in LDS
    __device__ __forceinline__ void begin(const MxTile &t, int n0) {
        constexpr int FIRST = C::ST > 2 ? 2 : 1;
#pragma unroll
        for (int j = 0; j < FIRST; ++j)
#pragma unroll
            for (int q = 0; q < C::WI; ++q) request(q, j, lds + j * C::STAGE);
        rows(t, n0);
        scales(0);
#pragma unroll
        for (int j = 0; j < C::ST - 1; ++j)
#pragma unroll
            for (int q = j < FIRST ? C::WI : 0; q < C::REQ; ++q) request(q, j, lds + j * C::STAGE);
        keep(0);
        wait_vmcnt<C::ST == 2 ? 0 : C::XI + (C::ST - 3) * C::REQ>();  // all but the second stage's activations and what came behind them
        wg_barrier();
    }
    // row r of the tile's weights: of which matrix, which row behind n0
    __device__ __forceinline__ static bool second(int r) { return C::GATED && (r >> 5 & 1); }
    __device__ __forceinline__ static int wrow(int r) { return C::GATED ? (r >> 6) * 32 + (r & 31) : r; }

    // which group comes in turn; behind the last one itself
    __device__ __forceinline__ int turned(int group) const { return group >= groups ? group : group + turn - (group + turn >= groups ? groups : 0); }
    // k of part `part` of a step
    __device__ __forceinline__ int first_k(int step, int part) const {
        const int pair = s0 / 2 + turned(step >> 1);  // (s0 is even)
        return pair * (2 * C::SK) + (step & 1) * (C::X8 ? C::SK : 64) + part * 128;
    }
    // What of a request lies behind the last row is beyond the buffer's range, which counts the scalar offset too; what lies behind a row's end, or in a step behind the
    // last one, is sent there.
    __device__ __forceinline__ void request(int q, int step, uint8_t *stage) const {
        const bool isw = q < C::WI;
        const int row = ((isw ? q : q - C::WI) * C::NW + wave) * (1024 / (isw ? C::WROW : 128)), height = isw ? C::TN : C::TM, part = row / height, r = row % height;  // (the wave's)
        const int k0 = first_k(step, part), each = isw || C::X8 ? 1 : 2;
        const bool indexed = C::GATED && !isw, surplus = !isw && !indexed && row >= C::TM * C::XPARTS;
        const uint32_t lane_off = isw ? wlane : xlane[indexed ? q - C::WI : 0];
        const uint32_t o = (isw ? wplace : xplace) < (kend - k0) * each && !surplus ? lane_off : kOut;
        const int soff = k0 * each + (isw ? wrow(r) * wbytes : indexed ? 0 : r * xbytes);
        const bool two = isw && C::GATED && second(r);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(isw ? (two ? w2rsrc : wrsrc) : xrsrc, (__attribute__((address_space(3))) void *)(stage + (q * C::NW + wave) * 1024), 16, o, soff,
                                                 0, 0);
    }
    // group: of two steps, counted from the part's first
    __device__ __forceinline__ void scales(int group) {
        const int g = s0 / 2 + turned(group), at = (g < whole ? g : whole > 0 ? whole - 1 : 0) * C::GE;
        typedef float group_t __attribute__((ext_vector_type(C::GE), aligned(4)));
        const group_t v = *(const __attribute__((address_space(1))) group_t *)(srow + at);
#pragma unroll
        for (int e = 0; e < C::GE; ++e) sv[e] = v[e];
    }
    __device__ __forceinline__ void keep(int group) const {
        float *const d = reinterpret_cast<float *>(lds + (tid < C::SROWS ? C::S_OFF + (group & 1) * C::S_GROUP + tid * 4 : C::DUMP + lane * 4));
        const int pitch = tid < C::SROWS ? C::SPITCH : 64, g = s0 / 2 + turned(group);
#pragma unroll
        for (int e = 0; e < C::GE; ++e) d[e * pitch] = g < whole ? sv[e] : tail[e];
    }
    // scale of row r (of SROWS) for block e of the group
    __device__ __forceinline__ float scale(int group, int e, int r) const {
        return *reinterpret_cast<const float *>(lds + C::S_OFF + (group & 1) * C::S_GROUP + (e * C::SPITCH + r) * 4);
    }
};

// ---- FP8 x.  A lane's part of a block of 16 rows: row l16, two pieces of 16 k of the step's block wk; of a result: activation row l16, n = 4 kg + 0..3
template <typename C>
__device__ __forceinline__ void sum_fp8(Source<C> &src, const MxTile &t, int n0, f32x4 (&acc)[2 * C::NB][2 * C::MB]) {
    constexpr int N = 2 * C::NB, M = 2 * C::MB, PAIRS = C::NB, ST = C::ST, LAG = 3, SW = C::GATED ? 2 : 1;
    const int lane = src.lane, wave = src.wave, l16 = lane & 15, kg = lane >> 4, wn = wave % C::WN, wm = wave / C::WN % C::WM, wk = wave / (C::WN * C::WM);
    uint8_t *const lds = src.lds;
#pragma unroll
    for (int a = 0; a < N; ++a)
#pragma unroll
        for (int b = 0; b < M; ++b) acc[a][b] = f32x4{0.f, 0.f, 0.f, 0.f};

    src.begin(t, n0);

    // (row r = 16 i + l16: key (r >> 1) & 7 = l16 >> 1)
    const uint32_t wl = (wk * C::TN + wn * C::NB * 32 + l16) * 128, xl = C::W_STAGE + (wk * C::TM + wm * C::MB * 32 + l16) * 128;
    // Pieces of 16 k: a read takes 16 lanes at a time, eight of l16's rows with an even kg and the other eight with the next kg; with pieces that differ in
    // the last bit alone they cover all banks (2 kg and 2 kg + 1 instead: two cycles for one)
    const uint32_t c = (kg >> 1) * 4 + (kg & 1), p0 = 16 * (c ^ (l16 >> 1)), p1 = 16 * ((c + 2) ^ (l16 >> 1));
    auto fragment = [&](const uint8_t *at) {
        const u32x4 lo = *reinterpret_cast<const u32x4 *>(at + p0), hi = *reinterpret_cast<const u32x4 *>(at + p1);
        return __builtin_bit_cast(i32x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    i32x8 wf[2][2], xf[M];
    float s[SW][M];
    auto read_w = [&](int pair, int j, int buf, const uint8_t *stage) { wf[buf][j] = fragment(stage + wl + (pair * 2 + j) * 2048); };
    auto read_x = [&](int b, const uint8_t *stage) { xf[b] = fragment(stage + xl + b * 2048); };
    float sw[SW], sx[M];  // of the next step
    auto read_s = [&](int step) {
        const int e = (step & 1) * C::WK + wk;
#pragma unroll
        for (int j = 0; j < SW; ++j) sw[j] = src.scale(step >> 1, e, C::TM + (C::GATED ? j : (wn * C::NB * 32) >> 7));
#pragma unroll
        for (int b = 0; b < M; ++b) sx[b] = src.scale(step >> 1, e, wm * C::MB * 32 + b * 16 + l16);
    };
    auto multiply_s = [&] {
#pragma unroll
        for (int b = 0; b < M; ++b)
#pragma unroll
            for (int j = 0; j < SW; ++j) s[j][b] = sx[b] * sw[j];
    };
    read_s(0);
#pragma unroll
    for (int b = 0; b < M; ++b) read_x(b, lds);
#pragma unroll
    for (int j = 0; j < 2; ++j) read_w(0, j, 0, lds);

    constexpr int NE = 2 * M, NP = PAIRS * NE, DB = LAG + 1;  // MFMAs of a pair of weight rows' blocks, of a step
    static_assert(NP % DB == 0 && LAG < NE, "results of a step in the same places, its scales used before the next ones are read");
    f32x4 d[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) d[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int b = 0; b < M; ++b)
#pragma unroll
        for (int j = 0; j < SW; ++j) s[j][b] = 0.f;
    auto add = [&](auto at_c) {  // the result of MFMA number at of a step
        constexpr int at = decltype(at_c)::value, pair = at / NE, a = 2 * pair + at % 2, b = at % NE / 2;
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[a][b][v] = __builtin_fmaf(d[at % DB][v], s[C::GATED ? pair & 1 : 0][b], acc[a][b][v]);
    };
    int slot = 0;
    // Step i, the parity of its registers (par).  In front of the last pair of blocks of weight rows, whose fragments are in registers, the wave waits for its part of
    // stage i + 1; behind the barrier everybody's is there and stage i has been read: step i + ST is requested into its place, one request behind an MFMA here and
    // there up to the next barrier, and the next step's first fragments are read beside the last pair's MFMAs, an activation fragment into the registers of the one
    // that both have used.
    constexpr int LATE = (PAIRS - 1) * NE;  // MFMAs of a step in front of its barrier
    auto step = [&](int i, auto par_c) {
        constexpr int par = decltype(par_c)::value;
        const int at_slot = ST == 2 ? par : slot;
        uint8_t *const cur = lds + at_slot * C::STAGE, *const nxt = lds + (at_slot + 1 == ST ? 0 : at_slot + 1) * C::STAGE;
        uint8_t *const prv = lds + (at_slot == 0 ? ST - 1 : at_slot - 1) * C::STAGE;
        auto pair = [&](auto pc) {
            constexpr int P = decltype(pc)::value, buf = (par * PAIRS + P) & 1;
            constexpr bool late = P == PAIRS - 1;
            if constexpr (late) {
                if constexpr (par == 1) src.keep((i + 1) >> 1);
                wait_vmcnt<(ST - 2) * C::REQ>();
                wg_barrier();
                if constexpr (par == 0) src.scales((i >> 1) + 1);
            }
            __builtin_amdgcn_sched_barrier(0);
            auto one = [&](auto ec) {
                constexpr int e = decltype(ec)::value, at = P * NE + e, j = e % 2, b = e / 2;
                d[at % DB] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf[buf][j], xf[b], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
                if constexpr (at == LAG) multiply_s();  // (the last results of the step before have been added)
                add(std::integral_constant<int, at >= LAG ? at - LAG : NP + at - LAG>{});
                if constexpr (!late) {
                    if constexpr (e == 0 || e == M) read_w(P + 1, e / M, buf ^ 1, cur);
                } else {
                    if constexpr (e == 0 || e == M) read_w(0, e / M, buf ^ 1, nxt);
                    if constexpr (j == 1) read_x(b, nxt);
                    if constexpr (e == NE - 1) read_s(i + 1);  // (behind multiply_s, which is at LAG < NE)
                }
                const int pos = at + (late ? -LATE : NP - LATE);
#pragma unroll
                for (int r = C::requested(pos, NP); r < C::requested(pos + 1, NP); ++r) src.request(r, late ? i + ST : i + ST - 1, late ? cur : prv);
                __builtin_amdgcn_sched_barrier(0);
            };
            each(one, std::make_integer_sequence<int, NE>{});
        };
        each(pair, std::make_integer_sequence<int, PAIRS>{});
        slot = slot + 1 == ST ? 0 : slot + 1;
    };
    // (the requests of step ST - 1 that a step before the first one would have made behind its barrier)
#pragma unroll
    for (int r = 0; r < C::requested(NP - LATE, NP); ++r) src.request(r, ST - 1, lds + (ST - 1) * C::STAGE);
    // (A step behind the last one works on zeros.  No branch inside the loop: the compiler would move MFMAs behind it, past the barrier.)
    // Of a SIMD's two waves one goes first, so that one's MFMAs meet the other's FMAs and reads: 4096 x 14336 x 4096 242 us instead of 249
    if (wave & 4) __builtin_amdgcn_s_setprio(1);
    for (int i = 0; i < src.steps; i += 2) {
        step(i, std::integral_constant<int, 0>{});
        step(i + 1, std::integral_constant<int, 1>{});
    }
    auto rest = [&](auto ec) { add(std::integral_constant<int, NP - LAG + decltype(ec)::value>{}); };
    each(rest, std::make_integer_sequence<int, LAG>{});
}

// ---- bf16 x.  A lane's part of a block of 32 rows: row l32; of the wave's 64 k of a step 32, in two pieces of 16; a slice is 8 of them, 16 bytes of x; of
// a result: activation row l32, n = 8 g + 4 kq + 0..3 for g = 0..3
template <typename C>
__device__ __forceinline__ void sum_bf16(Source<C> &src, const MxTile &t, int n0, f32x16 (&acc)[C::NB][C::MB]) {
    constexpr int NB = C::NB, MB = C::MB, ST = C::ST, SL = 4, AH = NB * MB < 8 ? 2 : 1, FB = 2 * AH;  // AH: how many slices ahead fragments are read
    const int lane = src.lane, wave = src.wave, l32 = lane & 31, kq = lane >> 5, wn = wave % C::WN, wm = wave / C::WN % C::WM, wk = wave / (C::WN * C::WM);
    uint8_t *const lds = src.lds;
    f32x16 d[NB][MB];  // the block's sums
#pragma unroll
    for (int a = 0; a < NB; ++a)
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[a][b][v] = d[a][b][v] = 0.f;

    src.begin(t, n0);

    // the lane's h-th piece of 16 values is 2 kq + h of the part's four; of x there are twice as many
    const uint32_t wkey = key<64>(l32), xkey = key<128>(l32);
    uint32_t xoff[SL], woff[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        woff[h] = (wk * C::TN + wn * NB * 32 + l32) * 64 + 16 * ((kq * 2 + h) ^ wkey);
#pragma unroll
        for (int g = 0; g < 2; ++g) xoff[2 * h + g] = C::W_STAGE + (wk * C::TM + wm * MB * 32 + l32) * 128 + 16 * ((kq * 4 + 2 * h + g) ^ xkey);
    }
    u32x4 xf[FB][MB], q[2][2][NB];  // activations; the weights' values of this step and the next
    bf16x8 wo[2][NB];
    float sw[2][NB];
    auto read = [&](int s, int f, int buf, const uint8_t *stage) { xf[buf][f] = *reinterpret_cast<const u32x4 *>(stage + xoff[s] + f * 4096); };
    auto read_step = [&](int step, int par, const uint8_t *stage) {  // what is read once per step
#pragma unroll
        for (int a = 0; a < NB; ++a) {
            const int row = C::GATED ? a & 1 : ((wn * NB + a) * 32) >> 7;
            sw[par][a] = src.scale(step >> 1, wk, row);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int a = 0; a < NB; ++a) q[par][h][a] = *reinterpret_cast<const u32x4 *>(stage + woff[h] + a * 32 * C::WROW);
    };
    auto dequant = [&](int s, int a, int par, int buf) {
        const u32x2 lo = fp8_to_bf16(q[par][s / 2][a][2 * (s % 2)]), hi = fp8_to_bf16(q[par][s / 2][a][2 * (s % 2) + 1]);
        wo[buf][a] = __builtin_bit_cast(bf16x8, u32x4{lo.x, lo.y, hi.x, hi.y});
    };
    read_step(0, 0, lds);
#pragma unroll
    for (int a = 0; a < NB; ++a) sw[1][a] = 0.f;
#pragma unroll
    for (int s = 0; s < AH; ++s)
#pragma unroll
        for (int f = 0; f < MB; ++f) read(s, f, s, lds);
#pragma unroll
    for (int a = 0; a < NB; ++a) dequant(0, a, 0, 0);
    int slot = 0;
    // Step i, the parity of its registers (par).  In front of slice SL - AH, whose fragments and the later ones' are in registers, the wave waits for its part of stage
    // i + 1; behind the barrier everybody's is there and stage i has been read: step i + ST is requested into its place, one request behind an MFMA here and there up
    // to the next barrier, and the next step's first fragments are read beside the last slices' MFMAs.
    constexpr int NE = NB * MB, NP = SL * NE, LATE = (SL - AH) * NE;  // MFMAs of a slice, of a step, of a step in front of its barrier
    auto step = [&](int i, auto par_c) {
        constexpr int par = decltype(par_c)::value;
        const int at_slot = ST == 2 ? par : slot;
        uint8_t *const cur = lds + at_slot * C::STAGE, *const nxt = lds + (at_slot + 1 == ST ? 0 : at_slot + 1) * C::STAGE;
        uint8_t *const prv = lds + (at_slot == 0 ? ST - 1 : at_slot - 1) * C::STAGE;
        auto slice = [&](auto sc) {
            constexpr int s = decltype(sc)::value, at = par * SL + s;  // (fragment buffers in turn over two steps)
            constexpr bool first = s == 0 && par == 0;                 // of a block
            if constexpr (s == SL - AH) {
                // (the first step of a group asks for the next group's scales, its last one puts them into LDS)
                if constexpr (par == 1) src.keep((i + 1) >> 1);
                wait_vmcnt<(ST - 2) * C::REQ>();
                wg_barrier();
                if constexpr (par == 0) src.scales((i >> 1) + 1);
                read_step(i + 1, par ^ 1, nxt);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                const int a = e / MB, b = e % MB;
                if constexpr (first) {  // (the scale of the block before)
#pragma unroll
                    for (int v = 0; v < 16; ++v) {
                        acc[a][b][v] = __builtin_fmaf(d[a][b][v], sw[par ^ 1][a], acc[a][b][v]);
                        d[a][b][v] = 0.f;
                    }
                }
                d[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wo[at & 1][a], __builtin_bit_cast(bf16x8, xf[at % FB][b]), d[a][b], 0, 0, 0);
#pragma unroll
                for (int f = e * MB / NE; f < (e + 1) * MB / NE; ++f) {
                    if constexpr (s + AH < SL) read(s + AH, f, (at + AH) % FB, cur);
                    else read(s + AH - SL, f, (at + AH) % FB, nxt);
                }
#pragma unroll
                for (int w = e * NB / NE; w < (e + 1) * NB / NE; ++w) {
                    if constexpr (s + 1 < SL) dequant(s + 1, w, par, (at + 1) & 1);
                    else dequant(0, w, par ^ 1, (at + 1) & 1);
                }
                constexpr bool late = s >= SL - AH;
                const int pos = s * NE + e + (late ? -LATE : NP - LATE);
#pragma unroll
                for (int r = C::requested(pos, NP); r < C::requested(pos + 1, NP); ++r) src.request(r, late ? i + ST : i + ST - 1, late ? cur : prv);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        each(slice, std::make_integer_sequence<int, SL>{});
        slot = slot + 1 == ST ? 0 : slot + 1;
    };
    // (the requests of step ST - 1 that a step before the first one would have made behind its barrier)
#pragma unroll
    for (int r = 0; r < C::requested(NP - LATE, NP); ++r) src.request(r, ST - 1, lds + (ST - 1) * C::STAGE);
    static_assert(2 * SL % FB == 0, "the buffers after two steps are those at the beginning");
    // (A step behind the last one works on zeros.  No branch inside the loop: the compiler would move MFMAs behind it, past the barrier.)
    for (int i = 0; i < src.steps; i += 2) {
        step(i, std::integral_constant<int, 0>{});
        step(i + 1, std::integral_constant<int, 1>{});
    }
#pragma unroll
    for (int a = 0; a < NB; ++a)
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[a][b][v] = __builtin_fmaf(d[a][b][v], sw[1][a], acc[a][b][v]);
}

// The tile t, n0 by MB blocks of rows per wave
template <typename C>
__device__ __forceinline__ void tile_body(const Fp8Product &p, const MxTile &t, int n0, uint8_t *lds) {
    constexpr int NB = C::NB, MB = C::MB, NO = C::GATED ? NB / 2 : NB, TO = C::TO;
    Source<C> src(p, t, n0, lds);
    const int tid = src.tid, lane = src.lane, wave = src.wave, wn = wave % C::WN, wm = wave / C::WN % C::WM, wk = wave / (C::WN * C::WM);
    // a block's 16 values of a lane as four quads of consecutive n: quad g is at activation row m(g), columns n(g) .. + 3 of the block
    f32x4 sum[NB][MB][4];
    if constexpr (C::X8) {
        f32x4 acc[2 * NB][2 * MB];
        sum_fp8<C>(src, t, n0, acc);
#pragma unroll
        for (int a = 0; a < NB; ++a)
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int g = 0; g < 4; ++g) sum[a][b][g] = acc[2 * a + g / 2][2 * b + g % 2];
    } else {
        f32x16 acc[NB][MB];
        sum_bf16<C>(src, t, n0, acc);
#pragma unroll
        for (int a = 0; a < NB; ++a)
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int g = 0; g < 4; ++g) sum[a][b][g] = f32x4{acc[a][b][4 * g], acc[a][b][4 * g + 1], acc[a][b][4 * g + 2], acc[a][b][4 * g + 3]};
    }
    auto quad_m = [&](int g) { return C::X8 ? g % 2 * 16 + (lane & 15) : lane & 31; };
    auto quad_n = [&](int g) { return C::X8 ? g / 2 * 16 + 4 * (lane >> 4) : 8 * g + 4 * (lane >> 5); };
    wait_vmcnt<0>();  // (the last requests, of zeros that nobody reads: no memory of this workgroup may be written once it has ended)
    if constexpr (C::WK > 1) {  // the sums of the waves along K, in their order
        __syncthreads();
        f32x4 *const red = reinterpret_cast<f32x4 *>(lds) + (size_t)(wm * C::WN + wn) * (C::WK - 1) * NB * MB * 256 + lane;
        if (wk > 0)
#pragma unroll
            for (int a = 0; a < NB; ++a)
#pragma unroll
                for (int b = 0; b < MB; ++b)
#pragma unroll
                    for (int g = 0; g < 4; ++g) red[(((wk - 1) * NB + a) * MB + b) * 256 + g * 64] = sum[a][b][g];
        __syncthreads();
        if (wk == 0)
#pragma unroll
            for (int k = 0; k < C::WK - 1; ++k)
#pragma unroll
                for (int a = 0; a < NB; ++a)
#pragma unroll
                    for (int b = 0; b < MB; ++b)
#pragma unroll
                        for (int g = 0; g < 4; ++g) sum[a][b][g] += red[((k * NB + a) * MB + b) * 256 + g * 64];
    }
    // ---- results
    f32x4 out[NO][MB][4];
#pragma unroll
    for (int a = 0; a < NO; ++a)
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int v = 0; v < 4; ++v) out[a][b][g][v] = C::GATED ? silu_mul(sum[2 * a][b][g][v], sum[2 * a + 1][b][g][v]) : sum[C::GATED ? 2 * a : a][b][g][v];
    if constexpr (C::H8) {
        // through LDS in fp32, 16 lanes to a row's block
        static_assert(C::WK == 1, "every wave has results");
        constexpr int PITCH = TO * 4 + 16;
        __syncthreads();
#pragma unroll
        for (int a = 0; a < NO; ++a)
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<f32x4 *>(lds + ((wm * MB + b) * 32 + quad_m(g)) * PITCH + ((wn * NO + a) * 32 + quad_n(g)) * 4) = out[a][b][g];
        __syncthreads();
        const int l = tid & 15, G = fp8_blocks(p.N);
        for (int m = tid >> 4; m < t.rows; m += C::T / 16) {  // (columns behind N are sums of zeros)
            const f32x4 lo = reinterpret_cast<const f32x4 *>(lds + m * PITCH)[2 * l], hi = reinterpret_cast<const f32x4 *>(lds + m * PITCH)[2 * l + 1];
            const float f[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
            const Fp8Scale c(max_of_16(absmax8(f)));
            const size_t row = (size_t)(t.row0 + m);
            if (l * 8 < src.nrows) *reinterpret_cast<u32x2 *>(p.h8 + row * p.N + n0 + l * 8) = c.values(f);
            if (l == 0) p.h8s[row * G + (n0 >> 7)] = c.scale;
        }
        return;
    }
    if (!p.y_bf16) {
        if (wk > 0) return;
        float *const y = reinterpret_cast<float *>(p.y) + (size_t)blockIdx.y * p.M * p.N;
        const bool quads = p.N % 4 == 0 && (reinterpret_cast<uintptr_t>(y) & 15) == 0;
#pragma unroll
        for (int a = 0; a < NO; ++a)
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int m = (wm * MB + b) * 32 + quad_m(g), n = n0 + (wn * NO + a) * 32 + quad_n(g);
                    if (m >= t.rows) continue;
                    float *const d = y + (size_t)(t.row0 + m) * p.N + n;
                    if (quads && n < p.N) *reinterpret_cast<f32x4 *>(d) = out[a][b][g];
                    else
#pragma unroll
                        for (int v = 0; v < 4; ++v)
                            if (n + v < p.N) d[v] = out[a][b][g][v];
                }
        return;
    }
    // through LDS, so that whole rows are stored
    __syncthreads();
    constexpr int PITCH = TO * 2 + 16;
    if (wk == 0)
#pragma unroll
        for (int a = 0; a < NO; ++a)
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 v = out[a][b][g];
                    *reinterpret_cast<u32x2 *>(lds + ((wm * MB + b) * 32 + quad_m(g)) * PITCH + ((wn * NO + a) * 32 + quad_n(g)) * 2) =
                        u32x2{pack_bf16_rne(v.x, v.y), pack_bf16_rne(v.z, v.w)};
                }
    __syncthreads();
    const int nrows = src.nrows;
    uint16_t *const y = reinterpret_cast<uint16_t *>(p.y) + (size_t)t.row0 * p.N + n0;
    if (p.N % 8 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0) {  // n0 is a multiple of 32: rows of whole pieces
        for (int i = tid; i < t.rows * (TO / 8); i += C::T) {
            const int m = i / (TO / 8), c = i % (TO / 8) * 8;
            if (c < nrows) *reinterpret_cast<u32x4 *>(y + (size_t)m * p.N + c) = *reinterpret_cast<const u32x4 *>(lds + m * PITCH + c * 2);
        }
    } else {
        for (int i = tid; i < t.rows * TO; i += C::T) {
            const int m = i / TO, c = i % TO;
            if (c < nrows) y[(size_t)m * p.N + c] = *reinterpret_cast<const uint16_t *>(lds + m * PITCH + c * 2);
        }
    }
}

template <bool X8, bool GATED, int WN, int WM, int WK, int NB, int MB, int SK, int ST>
__global__ __launch_bounds__(64 * WN * WM * WK) __attribute__((amdgpu_waves_per_eu(2, 2))) void fp8_tile_kernel(Fp8Product p) {
    typedef Cfg<X8, GATED, WN, WM, WK, NB, MB, SK, ST> C;
    constexpr int TM = C::TM, TO = C::TO;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    // Which tile: workgroup i runs on XCD i % 8; each XCD takes consecutive tiles, which go through 8 row tiles before the next columns, so
    // that what runs on it at one time shares rows and columns through its L2
    const int tiles_n = (p.N + TO - 1) / TO;
    int n0 = 0;
    auto take = [&](int tiles_m) {
        const int64_t total = (int64_t)tiles_m * tiles_n, per_xcd = (total + 7) >> 3, id = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
        if ((blockIdx.x >> 3) >= per_xcd || id >= total) return -1;
        const int band = (int)(id / (8 * tiles_n)), in = (int)(id % (8 * tiles_n)), high = tiles_m - band * 8 < 8 ? tiles_m - band * 8 : 8;
        n0 = in / high * TO;
        return band * 8 + in % high;
    };
    MxTile t;
    if (p.offsets) {
        t = MxTiles{p.offsets, p.E, p.M, TM}.place(p.clear_rest, take);
        if (t.group < 0) {
            mx_clear(p.y, p.y_bf16, p.N, t, n0, TO);
            return;
        }
    } else {
        const int tm = take((p.M + TM - 1) / TM);
        if (tm < 0) return;
        t = {0, tm * TM, p.M - tm * TM < TM ? p.M - tm * TM : TM, 0, 0};
    }
    t = {uniform(t.group), uniform(t.row0), uniform(t.rows), 0, 0};
    // A cut tile whose waves all share its rows takes as many blocks of 32 of them as it has; where two or four waves split them (WM) it works on all, on zeros behind the last
    if constexpr (WM == 1 && MB > 1) {
        if (t.rows <= 32) return tile_body<Cfg<X8, GATED, WN, WM, WK, NB, 1, SK, ST>>(p, t, n0, lds);
        if constexpr (MB > 2)
            if (t.rows <= 64) return tile_body<Cfg<X8, GATED, WN, WM, WK, NB, 2, SK, ST>>(p, t, n0, lds);
    }
    tile_body<C>(p, t, n0, lds);
}

template <bool X8, bool GATED, int WN, int WM, int WK, int NB, int MB, int SK, int ST>
static int launch(const Fp8Product &p, hipStream_t st) {
    typedef Cfg<X8, GATED, WN, WM, WK, NB, MB, SK, ST> C;
    const int64_t tm = p.offsets ? mx_most_tiles(p.M, p.E, C::TM) : mx_ceil(p.M, C::TM), tiles = tm * mx_ceil(p.N, C::TO);
    if (tiles > (1 << 22)) return fail(CHADQ_ERR_SHAPE, "fp8 product: M=%d N=%d are too many tiles", p.M, p.N);
    static std::atomic<bool> set[64];  // more LDS than the default limit: once per device
    int dev = 0;
    CHADQ_HIP(hipGetDevice(&dev));
    if (dev >= 64 || !set[dev].load()) {
        CHADQ_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(&fp8_tile_kernel<X8, GATED, WN, WM, WK, NB, MB, SK, ST>), hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS));
        if (dev < 64) set[dev].store(true);
    }
    hipLaunchKernelGGL((fp8_tile_kernel<X8, GATED, WN, WM, WK, NB, MB, SK, ST>), dim3((int)((tiles + 7) / 8 * 8), p.parts()), dim3(C::T), C::LDS, st, p);
    return hip_check(hipGetLastError(), "fp8 product launch");
}

}  // namespace f8t

// The requests' offsets are 32-bit, up to 256 rows from a tile's first, or (rows read through an index) from x's first.
bool fp8_tile_ok(const Fp8Product &p) {
    const int64_t row = p.xs ? p.K : (int64_t)p.K * 2;
    return (int64_t)p.K * 256 < INT32_MAX && row * 256 < INT32_MAX && (!p.rows || row * p.x_rows < INT32_MAX);
}

// Tiles with a P have four waves and half a compute unit's LDS: two workgroups to a unit, of which one computes while the other waits at its barrier, begins or ends.  us,
// 8-bit x, eight waves / four: 4096^3 92 / 70 at 128 x 128 and 132 / 94 at 128 x 64, but where there is one workgroup to a unit 79 / 103 (1000 x 4096 x 14336).
int fp8_tile_launch(const Fp8Product &p, int tile, hipStream_t st) {
    using namespace f8t;
    //                                                       WN WM WK NB MB SK ST
    if (p.w2) {
        if (p.xs) {
            if (tile == F8_256x64) return launch<true, true, 4, 2, 1, 2, 1, 128, 3>(p, st);
            return launch<true, true, 4, 2, 1, 2, 2, 128, 3>(p, st);
        }
        switch (tile) {
        case F8_128x64: return launch<false, true, 2, 2, 2, 2, 1, 128, 4>(p, st);
        case F8_128x64P: return launch<false, true, 2, 2, 1, 2, 1, 64, 4>(p, st);
        case F8_256x64: return launch<false, true, 4, 1, 2, 2, 2, 128, 3>(p, st);
        case F8_256x64P: return launch<false, true, 4, 1, 1, 2, 2, 64, 3>(p, st);
        case F8_128x128P: return launch<false, true, 2, 2, 1, 2, 2, 64, 3>(p, st);
        default: return launch<false, true, 4, 2, 1, 2, 2, 64, 4>(p, st);
        }
    }
    if (p.xs) {
        switch (tile) {
        case F8_64x32: return launch<true, false, 2, 1, 4, 1, 1, 512, 3>(p, st);
        case F8_64x64: return launch<true, false, 2, 1, 4, 1, 2, 512, 2>(p, st);
        case F8_128x64: return launch<true, false, 4, 1, 2, 1, 2, 256, 3>(p, st);
        case F8_128x64P: return launch<true, false, 2, 2, 1, 2, 1, 128, 3>(p, st);
        case F8_256x64: return launch<true, false, 8, 1, 1, 1, 2, 128, 3>(p, st);
        case F8_128x128: return launch<true, false, 2, 2, 2, 2, 2, 256, 2>(p, st);
        case F8_128x128P: return launch<true, false, 2, 2, 1, 2, 2, 128, 2>(p, st);
        case F8_256x128: return launch<true, false, 4, 2, 1, 2, 2, 128, 3>(p, st);
        default: return launch<true, false, 2, 4, 1, 4, 2, 128, 2>(p, st);
        }
    }
    switch (tile) {
    case F8_64x32: return launch<false, false, 2, 1, 4, 1, 1, 256, 4>(p, st);
    case F8_64x64: return launch<false, false, 2, 1, 4, 1, 2, 256, 3>(p, st);
    case F8_128x64: return launch<false, false, 4, 1, 2, 1, 2, 128, 4>(p, st);
    case F8_128x64P: return launch<false, false, 2, 2, 1, 2, 1, 64, 4>(p, st);
    case F8_256x64: return launch<false, false, 4, 1, 2, 2, 2, 128, 3>(p, st);
    case F8_256x64P: return launch<false, false, 4, 1, 1, 2, 2, 64, 3>(p, st);
    case F8_128x128: return launch<false, false, 2, 2, 2, 2, 2, 128, 3>(p, st);
    case F8_128x128P: return launch<false, false, 2, 2, 1, 2, 2, 64, 3>(p, st);
    default: return launch<false, false, 4, 2, 1, 2, 2, 64, 4>(p, st);
    }
}

}  // namespace chadq
