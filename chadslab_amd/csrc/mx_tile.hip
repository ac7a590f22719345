// Products of many rows on MXFP4 weights, x bf16 or MXFP4, one matrix or one per group of rows.
//
// A workgroup's WN x WM waves share a tile of TN weight rows x TM activation rows; a wave sums NB x MB blocks of 32 x 32.  The weights are the
// matrix cores' first operand, so that a lane holds four consecutive n of one activation row.
//   MXFP4 x  v_mfma_scale_f32_32x32x64_f8f6f4: both operands and their scale bytes go in as they are stored
//   bf16 x   the codes become bf16 with their scale, exactly (16 conversions per 32 codes), v_mfma_f32_32x32x16_bf16
// A step is BPS scale blocks along K.  Codes and activations go global -> LDS by DMA, ST stages, requests dealt to the waves in equal numbers and placed between
// the MFMAs; a piece past the end of a row or of the matrix is requested beyond the buffer's range and arrives as zeros, so nothing in the loop knows about
// edges.  Scales are 4 or 8 bytes of a row and step, at any alignment: a thread loads two steps' of a row, two steps ahead, and puts them into LDS.  16-byte
// pieces of a row are XOR-swizzled by the row so that the 16 rows that a read takes at a time cover all banks.  WK > 1: waves of a workgroup split the blocks of a
// step and add their sums at the end, so that a small tile too has eight waves to hide its reads.
//
// Measured, bf16 x: 48 x 14336 x 4096 16.2 us, 1000 x 4096 x 14336 109-114 us = 1.03-1.08 PFLOP/s, 4096^3 116-121 us = 1.14-1.18 PFLOP/s (a bf16 library product of 8192^3:
// 1.40); MXFP4 x: 4096^3 42-43 us = 3.2 PFLOP/s, 4096 x 14336 x 4096 156 us = 3.1 PFLOP/s.  Matrix cores busy: 54 % of the cycles of
// 1000 x 4096 x 14336, 39 % of 4096 x 14336 x 4096 with MXFP4 x.  bf16: the loop of 4096^3 without loads and conversions takes 71 us, at a clock that the power leaves.  MXFP4 x,
// 4096 x 4096 x 14336: 124 us (3.9 PFLOP/s); without the loop's requests 101, without its fragment reads 119, without both 94, the MFMAs alone 88 (5.5 PFLOP/s);
// at K = 4096 a tile's first requests and its result, 128 KB from each compute unit at once, are a quarter of the 43 us.  Small tiles: what a compute unit gets by
// DMA, 40-60 KB per us.  256 x 256 in steps of 128 k with three or four stages: 5-10 % slower.  Four blocks of columns to a wave for the bf16 256 x 128 tile, scale conversion once per block, and a branch round the scales' loads (the compiler moves
// MFMAs behind it) were no faster.
#include <cmath>
#include <type_traits>
#include <utility>

#include "mx.h"

namespace chadq {
namespace mxt {

template <bool X4, int WN, int WM, int WK, int NB, int MB, int BPS, int ST>
struct Cfg {
    static constexpr int NW = WN * WM * WK, T = 64 * NW, TN = 32 * NB * WN, TM = 32 * MB * WM;
    static constexpr int WROW = BPS * 16;                                 // bytes of a weight row per step
    static constexpr int XROW = X4 ? WROW : 128, XPARTS = X4 ? 1 : BPS / 2;  // of an activation row, in parts of at most 128
    static constexpr int W_STAGE = TN * WROW, X_STAGE = TM * XROW * XPARTS;
    // DMA instructions per wave and step, as many for each (what is too many of them for few rows fills a place nobody reads)
    static constexpr int WI = W_STAGE / (1024 * NW), XI = (X_STAGE + 1024 * NW - 1) / (1024 * NW), REQ = WI + XI, STAGE = W_STAGE + XI * 1024 * NW;
    static_assert(WI * 1024 * NW == W_STAGE && X_STAGE % 1024 == 0, "whole DMA instructions");
    static constexpr int SROWS = X4 ? TN + TM : TN, SPT = (SROWS + T - 1) / T;  // rows of scales per step, per thread
    static constexpr int GB = 2 * BPS, S_STAGE = SROWS * GB, S_OFF = ST * STAGE;  // a row's scales of two steps, loaded together
    static constexpr int HB = BPS / 2 / WK;                               // scale blocks of a lane and step
    static constexpr int SL = X4 ? HB : 4 * HB, AH = SL >= 4 && NB * MB < 8 ? 2 : 1;  // slices of a step; how far ahead fragments are read
    static_assert(HB * WK * 2 == BPS && SL >= AH, "each wave has whole blocks");
    static constexpr int DUMP = S_OFF + 2 * S_STAGE, OPER = DUMP + (SROWS % T ? 1024 : 0), RED = WN * WM * (WK - 1) * NB * MB * 4096;
    static constexpr int lds(int to) {  // to: result columns of a tile
        const int ep = TM * (to * 2 + 16), a = OPER > RED ? OPER : RED;
        return a > ep ? a : ep;
    }
    static_assert(BPS == 4 || BPS == 8, "scale bytes of a row and step: 4 or 8");
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

// The tile t, n0 by MB blocks of rows per wave
template <bool X4, bool GATED, int WN, int WM, int WK, int NB, int MB, int BPS, int ST>
__device__ __forceinline__ void tile_body(const MxProduct &p, const MxTile &t, int n0, uint8_t *lds) {
    typedef Cfg<X4, WN, WM, WK, NB, MB, BPS, ST> C;
    constexpr int TN = C::TN, TM = C::TM, TO = GATED ? TN / 2 : TN, NW = C::NW;  // TO: result columns
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, kq = lane >> 5, wn = wave % WN, wm = wave / WN % WM, wk = wave / (WN * WM);
    // K of this workgroup: the scale blocks of its part, from step s0 on
    const int G = p.K >> 5, s0 = p.part_k ? (int)blockIdx.y * (p.part_k / (32 * BPS)) : 0, gend = p.part_k && (s0 * BPS + p.part_k / 32) < G ? s0 * BPS + p.part_k / 32 : G;
    const int steps = (gend - s0 * BPS + BPS - 1) / BPS;

    // ---- requests
    const int wbytes = p.K >> 1, xbytes = X4 ? wbytes : p.K * 2;  // of a row
    const int nrows = p.N - n0 < TO ? p.N - n0 : TO;
    // row r of the tile's weights: of which matrix, which row behind n0
    auto second = [](int r) { return GATED && (r >> 5 & 1); };
    auto wrow = [](int r) { return GATED ? (r >> 6) * 32 + (r & 31) : r; };
    const size_t wfirst = (size_t)t.group * p.N + n0;
    auto weights = [&](const uint8_t *w) {
        return __builtin_amdgcn_make_buffer_rsrc(uniform(w + wfirst * wbytes), 0, uniform(nrows * wbytes), 0x00020000);
    };
    const __amdgpu_buffer_rsrc_t wrsrc = weights(p.w), w2rsrc = GATED ? weights(p.w2) : wrsrc;
    const __amdgpu_buffer_rsrc_t xrsrc = __builtin_amdgcn_make_buffer_rsrc(
        uniform(reinterpret_cast<const uint8_t *>(p.x) + (p.rows ? (size_t)0 : (size_t)t.row0 * xbytes)), 0, uniform((p.rows ? p.x_rows : t.rows) * xbytes), 0x00020000);
    constexpr uint32_t kOut = 0x80000000u;
    uint32_t off[C::REQ];
    int place[C::REQ];  // of the lane's piece in its row and step
#pragma unroll
    for (int q = 0; q < C::REQ; ++q) {
        if (q < C::WI) {
            constexpr int PPR = C::WROW / 16;
            const int r = (q * NW + wave) * (64 / PPR) + lane / PPR;
            place[q] = 16 * ((lane % PPR) ^ key<C::WROW>(r));
            off[q] = wrow(r) < nrows ? (uint32_t)wrow(r) * (uint32_t)wbytes + place[q] : kOut;
        } else {
            constexpr int PPR = C::XROW / 16;
            const int e = ((q - C::WI) * NW + wave) * (64 / PPR) + lane / PPR, r = e % TM;
            place[q] = e / TM * 128 + 16 * ((lane % PPR) ^ key<C::XROW>(r));
            const int src = r < t.rows ? (p.rows ? p.rows[t.row0 + r] : r) : 0;
            off[q] = r < t.rows && e < TM * C::XPARTS ? (uint32_t)src * (uint32_t)xbytes + place[q] : kOut;
        }
    }
    static_assert(!GATED || 1024 / C::WROW <= 32, "a DMA instruction's rows are of one block");
    auto request = [&](int q, int step, uint8_t *stage) {
        const bool isw = q < C::WI;
        const int soff = (s0 + step) * (isw ? C::WROW : C::XROW * C::XPARTS);
        const uint32_t o = soff + place[q] < gend * (isw || X4 ? 16 : 64) ? off[q] : kOut;
        const bool two = isw && GATED && second((q * NW + wave) * (1024 / C::WROW));
        __builtin_amdgcn_raw_ptr_buffer_load_lds(isw ? (two ? w2rsrc : wrsrc) : xrsrc, (__attribute__((address_space(3))) void *)(stage + (q * NW + wave) * 1024), 16, o, soff, 0,
                                                 0);
    };
    // scales: the thread's rows, GB bytes = two steps' (a group) at a time.  Those of the last group, if it is no whole one, are loaded byte by byte before the loop
    // (zeros behind the end of the row, where the activations are zeros too).  No branch: a thread without a row loads another one's and writes where nobody reads, and
    // so does the loop behind the last whole group.
    constexpr int GB = C::GB, GW = GB / 4;
    typedef __attribute__((ext_vector_type(GW))) uint32_t group_t;
    const int whole = G / GB;
    const uint8_t *srow[C::SPT];
    group_t sv[C::SPT], tail[C::SPT];
#pragma unroll
    for (int i = 0; i < C::SPT; ++i) {
        const int r = tid + i * C::T < C::SROWS ? tid + i * C::T : 0;
        const int n = wrow(r) < nrows ? wrow(r) : nrows - 1, m = r - TN < t.rows ? r - TN : t.rows - 1;
        srow[i] = !X4 || r < TN ? (second(r) ? p.w2s : p.ws) + (wfirst + n) * (size_t)G : p.xs + (size_t)(t.row0 + m) * G;
#pragma unroll
        for (int e = 0; e < GW; ++e) tail[i][e] = 0;
        if (G % GB)
#pragma unroll
            for (int b = 0; b < GB; ++b) tail[i][b / 4] |= (whole * GB + b < G ? (uint32_t)srow[i][whole * GB + b] : 0u) << (8 * (b % 4));
        if (whole == 0) srow[i] = p.w;  // (readable, for the loop)
    }
    auto scales = [&](int group) {
        const int g = s0 / 2 + group, at = (g < whole ? g : whole > 0 ? whole - 1 : 0) * GB;
#pragma unroll
        for (int i = 0; i < C::SPT; ++i) __builtin_memcpy(&sv[i], srow[i] + at, GB);
    };
    auto keep = [&](int group) {
#pragma unroll
        for (int i = 0; i < C::SPT; ++i) {
            const int r = tid + i * C::T;
            group_t v;
#pragma unroll
            for (int e = 0; e < GW; ++e) v[e] = s0 / 2 + group < whole ? sv[i][e] : tail[i][e];
            *reinterpret_cast<group_t *>(lds + (C::SROWS % C::T == 0 || r < C::SROWS ? C::S_OFF + (group & 1) * C::S_STAGE + r * GB : C::DUMP + lane * GB)) = v;
        }
    };

    f32x16 acc[NB][MB];
#pragma unroll
    for (int a = 0; a < NB; ++a)
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[a][b][v] = 0.f;

    scales(0);
#pragma unroll
    for (int j = 0; j < ST - 1; ++j)
#pragma unroll
        for (int r = 0; r < C::REQ; ++r) request(r, j, lds + j * C::STAGE);
    keep(0);
    wait_vmcnt<(ST - 2) * C::REQ>();
    wg_barrier();

    // ---- fragments.  The lane's block h of a step is kq * BPS / 2 + wk * HB + h; a slice is one of its blocks (MXFP4 x) or 8 k of it (bf16)
    const int blk0 = kq * (BPS / 2) + wk * C::HB;
    const uint32_t wkey = key<C::WROW>(l32), xkey = key<C::XROW>(l32);
    const uint32_t wl = (wn * NB * 32 + l32) * C::WROW, xl = C::W_STAGE + (wm * MB * 32 + l32) * C::XROW;
    const uint32_t sl = C::S_OFF + (wn * NB * 32 + l32) * GB + kq * (BPS / 2), xsl = C::S_OFF + (TN + wm * MB * 32 + l32) * GB + kq * (BPS / 2);
    constexpr int SL = C::SL, AH = C::AH, HB = C::HB, FB = 2 * AH;  // FB: fragment buffers
    u32x4 xf[FB][MB], wf[X4 ? FB : 1][X4 ? NB : 1];
    u32x4 q[2][X4 ? 1 : HB][X4 ? 1 : NB];  // bf16: the packed weights of this step and the next
    uint32_t ws[2][NB], xs[2][X4 ? MB : 1];
    bf16x8 wo[2][X4 ? 1 : NB];
    uint32_t xoff[SL], woff[HB];  // of a slice's fragment of the first activation block, of a block's weights
#pragma unroll
    for (int s = 0; s < SL; ++s) {
        const uint32_t piece = X4 ? blk0 + s : blk0 * 4 + s;  // of 16 bytes
        xoff[s] = xl + (X4 ? 0 : piece / 8 * (TM * 128)) + 16 * ((X4 ? piece : piece % 8) ^ xkey);
    }
#pragma unroll
    for (int h = 0; h < HB; ++h) woff[h] = wl + 16 * ((blk0 + h) ^ wkey);
    constexpr int NR = X4 ? NB + MB : MB;  // fragments of a slice: of the weights (MXFP4 x), of the activations
    auto read = [&](int s, int f, int buf, const uint8_t *stage) {
        if constexpr (X4) {
            if (f < NB) wf[buf][f] = *reinterpret_cast<const u32x4 *>(stage + woff[s] + f * 32 * C::WROW);
            else xf[buf][f - NB] = *reinterpret_cast<const u32x4 *>(stage + xoff[s] + (f - NB) * 32 * C::XROW);
        } else {
            xf[buf][f] = *reinterpret_cast<const u32x4 *>(stage + xoff[s] + f * 4096);
        }
    };
    auto read_step = [&](int step, int par, const uint8_t *stage) {  // what is read once per step
        const uint8_t *const sc = lds + (step >> 1 & 1) * C::S_STAGE + (step & 1) * BPS;
        auto word = [&](uint32_t at) {  // the wave's blocks first
            return (BPS == 8 ? *reinterpret_cast<const uint32_t *>(sc + at) : (uint32_t)*reinterpret_cast<const uint16_t *>(sc + at)) >> (8 * wk * HB);
        };
#pragma unroll
        for (int a = 0; a < NB; ++a) ws[par][a] = word(sl + a * 32 * GB);
        if constexpr (X4) {
#pragma unroll
            for (int b = 0; b < MB; ++b) xs[par][b] = word(xsl + b * 32 * GB);
        } else {
#pragma unroll
            for (int h = 0; h < HB; ++h)
#pragma unroll
                for (int a = 0; a < NB; ++a) q[par][h][a] = *reinterpret_cast<const u32x4 *>(stage + woff[h] + a * 32 * C::WROW);
        }
    };
    auto dequant = [&](int s, int a, int par, int buf) {
        if constexpr (!X4) wo[buf][a] = dequant8_mx(q[par][s / 4][a][s % 4], mx_scale((ws[par][a] >> (8 * (s / 4))) & 255u));
    };

    read_step(0, 0, lds);
#pragma unroll
    for (int s = 0; s < AH; ++s)
#pragma unroll
        for (int f = 0; f < NR; ++f) read(s, f, s, lds);
#pragma unroll
    for (int a = 0; a < NB; ++a) dequant(0, a, 0, 0);
    int slot = 0;
    // Step i, the parity of its registers (par).  In front of slice SL - AH, whose fragments and the later ones' are in registers, the wave waits for its part of stage
    // i + 1; behind the barrier everybody's is there and stage i has been read: step i + ST is requested into its place, one request behind an MFMA here and there up
    // to the next barrier, and the next step's first fragments are read beside the last slices' MFMAs.
    constexpr int NE = NB * MB, NP = SL * NE, LATE = (SL - AH) * NE;  // MFMAs of a slice, of a step, of a step in front of its barrier
    auto step = [&](int i, auto par_c) {
        constexpr int par = decltype(par_c)::value;
        uint8_t *const cur = lds + slot * C::STAGE, *const nxt = lds + (slot + 1 == ST ? 0 : slot + 1) * C::STAGE;
        uint8_t *const prv = lds + (slot == 0 ? ST - 1 : slot - 1) * C::STAGE;
        auto slice = [&](auto sc) {
            constexpr int s = decltype(sc)::value, at = par * SL + s;  // (fragment buffers in turn over two steps)
            if constexpr (s == SL - AH) {
                // (the first step of a group asks for the next group's scales, its last one puts them into LDS)
                if constexpr (par == 1) keep((i + 1) >> 1);
                wait_vmcnt<(ST - 2) * C::REQ>();
                wg_barrier();
                if constexpr (par == 0) scales((i >> 1) + 1);
                read_step(i + 1, par ^ 1, nxt);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                const int a = e / MB, b = e % MB;
                if constexpr (X4)
                    acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(wf[at % FB][a]), mx_operand(xf[at % FB][b]), acc[a][b], 4, 4, s, (int)ws[par][a], s,
                                                                                (int)xs[par][b]);
                else
                    acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wo[at & 1][a], __builtin_bit_cast(bf16x8, xf[at % FB][b]), acc[a][b], 0, 0, 0);
#pragma unroll
                for (int f = e * NR / NE; f < (e + 1) * NR / NE; ++f) {
                    if constexpr (s + AH < SL) read(s + AH, f, (at + AH) % FB, cur);
                    else read(s + AH - SL, f, (at + AH) % FB, nxt);
                }
#pragma unroll
                for (int d = e * NB / NE; d < (e + 1) * NB / NE; ++d) {
                    if constexpr (s + 1 < SL) dequant(s + 1, d, par, (at + 1) & 1);
                    else dequant(0, d, par ^ 1, (at + 1) & 1);
                }
                constexpr bool late = s >= SL - AH;
                const int pos = s * NE + e + (late ? -LATE : NP - LATE);
#pragma unroll
                for (int r = pos * C::REQ / NP; r < (pos + 1) * C::REQ / NP; ++r) request(r, late ? i + ST : i + ST - 1, late ? cur : prv);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        each(slice, std::make_integer_sequence<int, SL>{});
        slot = slot + 1 == ST ? 0 : slot + 1;
    };
    // (the requests of step ST - 1 that a step before the first one would have made behind its barrier)
#pragma unroll
    for (int r = 0; r < (NP - LATE) * C::REQ / NP; ++r) request(r, ST - 1, lds + (ST - 1) * C::STAGE);
    static_assert(2 * SL % FB == 0, "the buffers after two steps are those at the beginning");
    // (A step behind the last one works on zeros.  No branch inside the loop: the compiler would move MFMAs behind it, past the barrier.)
    for (int i = 0; i < steps; i += 2) {
        step(i, std::integral_constant<int, 0>{});
        step(i + 1, std::integral_constant<int, 1>{});
    }
    wait_vmcnt<0>();  // (the last requests, of zeros that nobody reads: no memory of this workgroup may be written once it has ended)
    if constexpr (WK > 1) {  // the sums of the waves along K, in their order
        __syncthreads();
        f32x4 *const red = reinterpret_cast<f32x4 *>(lds) + (size_t)(wm * WN + wn) * (WK - 1) * NB * MB * 256 + lane;
        if (wk > 0)
#pragma unroll
            for (int a = 0; a < NB; ++a)
#pragma unroll
                for (int b = 0; b < MB; ++b)
#pragma unroll
                    for (int g = 0; g < 4; ++g)
                        red[(((wk - 1) * NB + a) * MB + b) * 256 + g * 64] = f32x4{acc[a][b][4 * g], acc[a][b][4 * g + 1], acc[a][b][4 * g + 2], acc[a][b][4 * g + 3]};
        __syncthreads();
        if (wk == 0)
#pragma unroll
            for (int k = 0; k < WK - 1; ++k)
#pragma unroll
                for (int a = 0; a < NB; ++a)
#pragma unroll
                    for (int b = 0; b < MB; ++b)
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const f32x4 v = red[((k * NB + a) * MB + b) * 256 + g * 64];
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[a][b][4 * g + e] += v[e];
                        }
    }
    // ---- results.  A lane's values of a block: activation row l32, n = 8 g + 4 kq + 0..3 for g = 0..3
    constexpr int NO = GATED ? NB / 2 : NB;
    static_assert(!GATED || NB % 2 == 0, "gate and up blocks side by side");
    f32x4 out[NO][MB][4];
#pragma unroll
    for (int a = 0; a < NO; ++a)
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v) out[a][b][v / 4][v % 4] = GATED ? silu_mul(acc[2 * a][b][v], acc[2 * a + 1][b][v]) : acc[GATED ? 2 * a : a][b][v];
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
                    const int m = (wm * MB + b) * 32 + l32, n = n0 + (wn * NO + a) * 32 + 8 * g + 4 * kq;
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
                *reinterpret_cast<u32x2 *>(lds + ((wm * MB + b) * 32 + l32) * PITCH + ((wn * NO + a) * 32 + 8 * g + 4 * kq) * 2) =
                    u32x2{pack_bf16_rne(v.x, v.y), pack_bf16_rne(v.z, v.w)};
            }
    __syncthreads();
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

template <bool X4, bool GATED, int WN, int WM, int WK, int NB, int MB, int BPS, int ST>
__global__ __launch_bounds__(64 * WN * WM * WK) __attribute__((amdgpu_waves_per_eu(WN * WM * WK / 4, WN * WM * WK / 4))) void mx_tile_kernel(MxProduct p) {
    typedef Cfg<X4, WN, WM, WK, NB, MB, BPS, ST> C;
    constexpr int TM = C::TM, TO = GATED ? C::TN / 2 : C::TN;
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
    // A cut tile takes as many blocks of 32 rows as it has
    if constexpr (WM == 1 && MB > 1) {
        if (t.rows <= 32) return tile_body<X4, GATED, WN, WM, WK, NB, 1, BPS, ST>(p, t, n0, lds);
        if constexpr (MB > 2)
            if (t.rows <= 64) return tile_body<X4, GATED, WN, WM, WK, NB, 2, BPS, ST>(p, t, n0, lds);
    }
    tile_body<X4, GATED, WN, WM, WK, NB, MB, BPS, ST>(p, t, n0, lds);
}

template <bool X4, bool GATED, int WN, int WM, int WK, int NB, int MB, int BPS, int ST>
static int launch(const MxProduct &p, hipStream_t st) {
    typedef Cfg<X4, WN, WM, WK, NB, MB, BPS, ST> C;
    constexpr int TO = GATED ? C::TN / 2 : C::TN, LDS = C::lds(TO);
    static_assert(LDS <= 163840, "LDS of a compute unit");
    const int64_t tm = p.offsets ? mx_most_tiles(p.M, p.E, C::TM) : mx_ceil(p.M, C::TM), tiles = tm * mx_ceil(p.N, TO);
    if (tiles > (1 << 22)) return fail(CHADQ_ERR_SHAPE, "mxfp4 product: M=%d N=%d are too many tiles", p.M, p.N);
    static std::atomic<bool> set[64];  // more LDS than the default limit: once per device
    int dev = 0;
    CHADQ_HIP(hipGetDevice(&dev));
    if (dev >= 64 || !set[dev].load()) {
        CHADQ_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(&mx_tile_kernel<X4, GATED, WN, WM, WK, NB, MB, BPS, ST>), hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
        if (dev < 64) set[dev].store(true);
    }
    hipLaunchKernelGGL((mx_tile_kernel<X4, GATED, WN, WM, WK, NB, MB, BPS, ST>), dim3((int)((tiles + 7) / 8 * 8), p.parts()), dim3(C::T), LDS, st, p);
    return hip_check(hipGetLastError(), "mxfp4 product launch");
}

}  // namespace mxt

// The requests' offsets are 32-bit, up to 256 rows from a tile's first, or (rows read through an index) from x's first.
bool mx_tile_ok(const MxProduct &p) {
    const int64_t row = p.xs ? p.K / 2 : (int64_t)p.K * 2;
    return row * 256 < INT32_MAX && (!p.rows || row * p.x_rows < INT32_MAX);
}

// ---- which tile, and K in how many parts
enum Tile { T64x32, T64x64, T128x64, T256x64, T128x128, T256x128, T256x256, T256x96, T128x96, T128x32, TILES };  // weight rows x activation rows

int mx_tile_launch(const MxProduct &p, int tile, hipStream_t st) {
    using namespace mxt;
    //                                                       WN WM WK NB MB BPS ST
    if (p.w2) {
        switch (tile) {
        case T128x32: return launch<false, true, 2, 1, 4, 2, 1, 8, 4>(p, st);
        case T128x64: return launch<false, true, 2, 1, 4, 2, 2, 8, 3>(p, st);
        case T256x64: return launch<false, true, 4, 1, 2, 2, 2, 4, 4>(p, st);
        case T256x96: return launch<false, true, 4, 1, 2, 2, 3, 4, 3>(p, st);
        default: return launch<false, true, 4, 2, 1, 2, 2, 4, 3>(p, st);
        }
    }
    if (p.xs) {
        switch (tile) {
        case T64x32: return launch<true, false, 2, 1, 4, 1, 1, 8, 6>(p, st);
        case T64x64: return launch<true, false, 2, 1, 4, 1, 2, 8, 6>(p, st);
        case T128x64: return launch<true, false, 4, 1, 2, 1, 2, 8, 6>(p, st);
        case T256x64: return launch<true, false, 4, 1, 2, 2, 2, 8, 3>(p, st);
        case T256x96: return launch<true, false, 4, 1, 2, 2, 3, 8, 3>(p, st);
        case T128x96: return launch<true, false, 4, 1, 2, 1, 3, 8, 4>(p, st);
        case T128x128: return launch<true, false, 2, 2, 2, 2, 2, 8, 4>(p, st);
        case T256x128: return launch<true, false, 4, 2, 1, 2, 2, 8, 3>(p, st);
        default: return launch<true, false, 2, 4, 1, 4, 2, 8, 2>(p, st);
        }
    }
    switch (tile) {
    case T64x32: return launch<false, false, 2, 1, 4, 1, 1, 8, 5>(p, st);
    case T64x64: return launch<false, false, 2, 1, 4, 1, 2, 8, 3>(p, st);
    case T128x64: return launch<false, false, 4, 1, 2, 1, 2, 4, 5>(p, st);
    case T256x64: return launch<false, false, 4, 1, 2, 2, 2, 4, 4>(p, st);
    case T256x96: return launch<false, false, 4, 1, 2, 2, 3, 4, 3>(p, st);
    case T128x96: return launch<false, false, 4, 1, 2, 1, 3, 4, 4>(p, st);
    case T128x128: return launch<false, false, 2, 2, 2, 2, 2, 4, 3>(p, st);
    default: return launch<false, false, 4, 2, 1, 2, 2, 4, 3>(p, st);
    }
}

// Time of a product by tile: `start` us once, and for each round of the compute units' workgroups `round` us and `few` (64 workgroups, at the clock that they leave) to
// `full` (256) us per 1024 k.  Measured at 64, 256 and 512 workgroups and K = 1024 and 4096.
struct TileTime {
    int tn, tm;
    float start, round, few, full;
};
static const TileTime kBf16[TILES] = {{64, 32, 1.5f, 2.7f, 1.46f, 1.55f},   {64, 64, 1.7f, 3.0f, 2.21f, 2.35f},  {128, 64, 1.4f, 1.8f, 4.82f, 5.1f},
                                      {256, 64, 1.7f, 2.3f, 7.31f, 7.85f},  {128, 128, 2.4f, 2.5f, 6.07f, 7.5f}, {256, 128, 0.6f, 4.7f, 9.29f, 13.2f},
                                      {256, 256, 0.f, 1e9f, 0.f, 0.f},      {256, 96, 2.3f, 3.1f, 8.0f, 10.5f},  {128, 96, 2.8f, 2.0f, 4.33f, 6.05f},
                                      {128, 32, 1.7f, 3.0f, 3.0f, 3.2f}};
static const TileTime kMx[TILES] = {{64, 32, 1.5f, 2.5f, 1.33f, 1.31f},  {64, 64, 1.4f, 3.2f, 1.26f, 1.29f},  {128, 64, 1.6f, 2.5f, 2.88f, 2.5f},
                                    {256, 64, 1.7f, 2.3f, 4.54f, 4.15f}, {128, 128, 2.2f, 3.0f, 3.21f, 3.1f}, {256, 128, 3.0f, 2.5f, 5.05f, 5.15f},
                                    {256, 256, 1.8f, 6.8f, 7.34f, 8.1f}, {256, 96, 2.4f, 3.3f, 5.0f, 4.6f},   {128, 96, 2.1f, 2.9f, 3.05f, 2.77f},
                                    {128, 32, 0.f, 1e9f, 0.f, 0.f}};

static MxTilePick pick(int M, int N, int K, int E, bool x_mx, bool gated, int most_parts) {
    MxTilePick best = {T128x128, 0};
    float least = 1e30f;
    for (int i = 0; i < TILES; ++i) {
        const TileTime &t = (x_mx ? kMx : kBf16)[i];
        const int tn = gated ? t.tn / 2 : t.tn;
        // (gated: 128 x 96 and 128 x 128 were up to 1.45x behind the fastest and never it; 128 x 32 is their tile for few rows or columns)
        if (t.round > 1e8f || (gated ? t.tn < 128 || i == T128x96 || i == T128x128 : i == T128x32)) continue;
        // rows by group: between the tiles of groups of one size and those of exponentially distributed sizes
        const float mean = (float)M / E > 1.f ? (float)M / E : 1.f, hit = E * (1.f - expf(-(float)M / E)), even = mean / t.tm + 0.3f;
        const float tm = E > 1 ? hit * 0.5f * ((even > 1.f ? even : 1.f) + 1.f / (1.f - expf(-t.tm / mean))) : (float)mx_ceil(M, t.tm);
        const float tiles = tm * mx_ceil(N, tn);
        for (int parts = 1; parts <= most_parts; ++parts) {
            const int part_k = parts > 1 ? ((K + parts - 1) / parts + 511) / 512 * 512 : K;
            if (parts > 1 && (part_k < 1024 || (int64_t)part_k * (parts - 1) >= K)) continue;
            const float wgs = tiles * parts, full = wgs >= 256.f ? 1.f : wgs <= 64.f ? 0.f : (wgs - 64.f) / 192.f;
            // (by group: a workgroup finds its tile first; the groups' tiles end unevenly)
            const float rounds = E > 1 && wgs > 256.f ? wgs / 256.f + 0.6f : ceilf(wgs / 256.f), round = E > 1 ? t.round + 2.f : t.round;
            // (a cut tile one wave high takes fewer blocks of rows; one block costs this share of two or three)
            const float one = E == 1 ? 1.f : t.tm == 96 ? 0.6f : t.tm == 64 ? 0.8f : 1.f, rows = (float)M / (tm * t.tm);
            float us = t.start + rounds * (round + (t.few + (t.full - t.few) * full) * (one + (1.f - one) * (rows < 1.f ? rows : 1.f)) * (part_k / 1024.f));
            if (parts > 1) us += 3.f + (8.f * parts + 2.f) * M * (float)N * 2.5e-7f;  // the sums written, read again and joined by another launch
            if (us < least * (parts > 1 ? 0.95f : 1.f)) {
                least = us;
                best = {i, parts > 1 ? part_k : 0};
            }
        }
    }
    return best;
}

MxTilePick mx_tile_pick(const MxProduct &p, int most_parts) { return pick(p.M, p.N, p.K, p.offsets ? p.E : 1, p.xs != nullptr, p.w2 != nullptr, most_parts); }


// y = the parts' sums, added in their order; four values to a thread where the rows allow
__global__ __launch_bounds__(256) void mx_join_kernel(const float *__restrict__ part, void *__restrict__ y, int64_t n, int parts, bool y_bf16, bool quads) {
    const int64_t stride = (int64_t)gridDim.x * 256, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (quads) {
        for (int64_t i = at; i < n / 4; i += stride) {
            f32x4 v = reinterpret_cast<const f32x4 *>(part)[i];
            for (int k = 1; k < parts; ++k) v += reinterpret_cast<const f32x4 *>(part + k * n)[i];
            if (y_bf16) reinterpret_cast<u32x2 *>(y)[i] = u32x2{pack_bf16_rne(v.x, v.y), pack_bf16_rne(v.z, v.w)};
            else reinterpret_cast<f32x4 *>(y)[i] = v;
        }
    } else {
        for (int64_t i = at; i < n; i += stride) {
            float v = part[i];
            for (int k = 1; k < parts; ++k) v += part[k * n + i];
            store_sum(reinterpret_cast<float *>(y), i, v, y_bf16);
        }
    }
}

int mx_join_launch(const float *part, void *y, int64_t n, int parts, bool y_bf16, hipStream_t st) {
    const bool quads = n % 4 == 0 && aligned16(y);
    const int64_t items = quads ? n / 4 : n;
    hipLaunchKernelGGL(mx_join_kernel, dim3((int)(items < 2048 * 256 ? (items + 255) / 256 : 2048)), dim3(256), 0, st, part, y, n, parts, y_bf16, quads);
    return hip_check(hipGetLastError(), "join launch");
}

// The product in its parts of K: fp32 sums to `part`, joined into y
int mx_tile_parts_launch(const MxProduct &p, int tile, float *part, hipStream_t st) {
    MxProduct q = p;
    q.y = part;
    q.y_bf16 = false;
    const int rc = mx_tile_launch(q, tile, st);
    if (rc) return rc;
    return mx_join_launch(part, p.y, (int64_t)p.M * p.N, q.parts(), p.y_bf16, st);
}

}  // namespace chadq
