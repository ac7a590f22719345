// Products of many rows on MXFP4 weights, x bf16 or MXFP4, one matrix or one per group of rows.
//
// A workgroup's WN x WM waves share a tile of TN weight rows x TM activation rows; a wave sums NB x MB blocks of 32 x 32.  The weights are the
// matrix cores' first operand, so that a lane holds four consecutive n of one activation row.
//   MXFP4 x  v_mfma_scale_f32_32x32x64_f8f6f4: both operands and their scale bytes go in as they are stored
//   bf16 x   the codes become bf16 with their scale, exactly (16 conversions per 32 codes), v_mfma_f32_32x32x16_bf16
// A step is BPS scale blocks along K.  Codes and activations go global -> LDS by DMA, ST stages, requests dealt to the waves in equal numbers; a
// piece past the end of a row or of the matrix is requested beyond the buffer's range and arrives as zeros, so nothing in the loop knows about
// edges.  Scales are 4 or 8 bytes of a row and step, at any alignment: one thread loads those of a row a step ahead and puts them into LDS.  16-byte pieces of
// a row are XOR-swizzled by the row so that the 16 rows that a read takes at a time cover all banks.
#include <type_traits>

#include "mx.h"

namespace chadq {
namespace mxt {

template <bool X4, int WN, int WM, int NB, int MB, int BPS, int ST>
struct Cfg {
    static constexpr int NW = WN * WM, T = 64 * NW, TN = 32 * NB * WN, TM = 32 * MB * WM;
    static constexpr int WROW = BPS * 16;                                 // bytes of a weight row per step
    static constexpr int XROW = X4 ? WROW : 128, XPARTS = X4 ? 1 : BPS / 2;  // of an activation row, in parts of at most 128
    static constexpr int W_STAGE = TN * WROW, X_STAGE = TM * XROW * XPARTS, STAGE = W_STAGE + X_STAGE;
    static constexpr int WI = W_STAGE / (1024 * NW), XI = X_STAGE / (1024 * NW), REQ = WI + XI;  // DMA instructions per wave and step
    static_assert(WI * 1024 * NW == W_STAGE && XI * 1024 * NW == X_STAGE, "the same number of whole DMA instructions for each wave");
    static constexpr int SROWS = X4 ? TN + TM : TN, SPT = (SROWS + T - 1) / T;  // rows of scales per step, per thread
    static constexpr int S_STAGE = SROWS * BPS, S_OFF = ST * STAGE;
    static constexpr int OPER = ST * STAGE + 2 * S_STAGE;
    static constexpr int lds(int to) { return OPER > TM * (to * 2 + 16) ? OPER : TM * (to * 2 + 16); }  // to: result columns of a tile
    static_assert(BPS == 4 || BPS == 8, "scale bytes of a row and step: 4 or 8");
};

// how the 16-byte pieces of row r are permuted: rows of 64 bytes, four of them to the banks, or of 128, two
template <int ROW>
__device__ __forceinline__ int key(int r) {
    return ROW == 64 ? (r >> 2) & 3 : (r >> 1) & 7;
}

template <bool X4, bool GATED, int WN, int WM, int NB, int MB, int BPS, int ST>
__global__ __launch_bounds__(64 * WN * WM) __attribute__((amdgpu_waves_per_eu(WN * WM / 4, WN * WM / 4))) void mx_tile_kernel(MxProduct p) {
    typedef Cfg<X4, WN, WM, NB, MB, BPS, ST> C;
    constexpr int TN = C::TN, TM = C::TM, TO = GATED ? TN / 2 : TN, NW = C::NW;  // TO: result columns
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31, kq = lane >> 5, wn = wave % WN, wm = wave / WN;
    const int G = p.K >> 5, steps = (G + BPS - 1) / BPS;

    // ---- which tile: workgroup i runs on XCD i % 8; each XCD takes consecutive tiles, which go through 8 row tiles before the next columns, so
    // that what runs on it at one time shares rows and columns through its L2
    const int tiles_n = (p.N + TO - 1) / TO;
    const MxTiles groups = {p.offsets, p.E, p.M, TM};
    const int tiles_m = p.offsets ? groups.count(p.clear_rest) : (p.M + TM - 1) / TM;
    const int64_t total = (int64_t)tiles_m * tiles_n, per_xcd = (total + 7) >> 3, id = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per_xcd || id >= total) return;
    const int band = (int)(id / (8 * tiles_n)), in = (int)(id % (8 * tiles_n)), high = tiles_m - band * 8 < 8 ? tiles_m - band * 8 : 8;
    const int tm = band * 8 + in % high, n0 = in / high * TO;
    MxTile t = {0, tm * TM, p.M - tm * TM < TM ? p.M - tm * TM : TM, 0, 0};
    if (p.offsets) {
        t = groups.find(tm);
        if (t.group < 0) {
            mx_clear(p.y, p.y_bf16, p.N, t, n0, TO);
            return;
        }
    }

    // ---- requests
    const int wbytes = p.K >> 1, xbytes = X4 ? wbytes : p.K * 2;  // of a row
    const int nrows = p.N - n0 < TO ? p.N - n0 : TO;
    // row r of the tile's weights: of which matrix, which row behind n0
    auto second = [](int r) { return GATED && (r >> 5 & 1); };
    auto wrow = [](int r) { return GATED ? (r >> 6) * 32 + (r & 31) : r; };
    const size_t wfirst = (size_t)t.group * p.N + n0;
    auto weights = [&](const uint8_t *w) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(w) + wfirst * wbytes, 0, nrows * wbytes, 0x00020000);
    };
    const __amdgpu_buffer_rsrc_t wrsrc = weights(p.w), w2rsrc = GATED ? weights(p.w2) : wrsrc;
    const __amdgpu_buffer_rsrc_t xrsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t *>(reinterpret_cast<const uint8_t *>(p.x)) + (p.rows ? (size_t)0 : (size_t)t.row0 * xbytes), 0, p.rows ? p.x_rows * xbytes : t.rows * xbytes, 0x00020000);
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
            off[q] = r < t.rows ? (uint32_t)src * (uint32_t)xbytes + place[q] : kOut;
        }
    }
    static_assert(!GATED || C::WROW == 64 || C::WROW == 128, "a DMA instruction's rows are of one block");
    auto request = [&](int step, uint8_t *stage) {
#pragma unroll
        for (int q = 0; q < C::REQ; ++q) {
            const bool isw = q < C::WI;
            const int soff = step * (isw ? C::WROW : C::XROW * C::XPARTS);
            const uint32_t o = soff + place[q] < (isw ? wbytes : xbytes) ? off[q] : kOut;
            const bool two = isw && GATED && second((q * NW + wave) * (1024 / C::WROW));
            __builtin_amdgcn_raw_ptr_buffer_load_lds(isw ? (two ? w2rsrc : wrsrc) : xrsrc, (__attribute__((address_space(3))) void *)(stage + (q * NW + wave) * 1024), 16, o, soff,
                                                     0, 0);
        }
    };
    // scales: the thread's rows
    const uint8_t *srow[C::SPT];
#pragma unroll
    for (int i = 0; i < C::SPT; ++i) {
        const int r = tid + i * C::T;
        const int n = wrow(r) < nrows ? wrow(r) : nrows - 1, m = r - TN < t.rows ? r - TN : t.rows - 1;
        srow[i] = !X4 || r < TN ? (second(r) ? p.w2s : p.ws) + (wfirst + n) * (size_t)G : p.xs + (size_t)(t.row0 + m) * G;
    }
    MxScales<BPS> sv[C::SPT];
    auto scales = [&](int step) {
#pragma unroll
        for (int i = 0; i < C::SPT; ++i)
            if (C::SROWS % C::T == 0 || tid + i * C::T < C::SROWS) {
                if (G >= BPS) {
                    sv[i].load(srow[i], step * BPS, G);
                } else {  // K < 32 BPS
                    sv[i].raw = 0;
                    sv[i].cut = 0;
                    for (int b = 0; b < G; ++b) sv[i].raw |= (typename MxScales<BPS>::bytes_t)srow[i][b] << (8 * b);
                }
            }
    };
    auto keep = [&](int step) {
#pragma unroll
        for (int i = 0; i < C::SPT; ++i)
            if (C::SROWS % C::T == 0 || tid + i * C::T < C::SROWS) {
                *reinterpret_cast<typename MxScales<BPS>::bytes_t *>(lds + C::S_OFF + (step & 1) * C::S_STAGE + (tid + i * C::T) * BPS) = sv[i].get();
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
    for (int j = 0; j < ST - 1; ++j) request(j, lds + j * C::STAGE);
    keep(0);
    int slot = 0;
    for (int i = 0; i < steps; ++i) {
        wait_vmcnt<(ST - 2) * C::REQ>();     // the wave's part of stage i is there
        wg_barrier();                        // everybody's, and the scales; stage i - 1 has been read
        const uint8_t *const cur = lds + slot * C::STAGE, *const sc = lds + C::S_OFF + (i & 1) * C::S_STAGE;
        scales(i + 1);
        request(i + ST - 1, lds + (slot == 0 ? ST - 1 : slot - 1) * C::STAGE);
        const uint8_t *const wl = cur + (wn * NB * 32 + l32) * C::WROW, *const sl = sc + (wn * NB * 32 + l32) * BPS + kq * (BPS / 2);
        const int wkey = key<C::WROW>(l32), xkey = key<C::XROW>(l32);
        const uint8_t *const xl = cur + C::W_STAGE + (wm * MB * 32 + l32) * C::XROW;
        uint32_t ws[NB];
#pragma unroll
        for (int a = 0; a < NB; ++a) ws[a] = BPS == 8 ? *reinterpret_cast<const uint32_t *>(sl + a * 32 * BPS) : *reinterpret_cast<const uint16_t *>(sl + a * 32 * BPS);
        if constexpr (X4) {
            uint32_t xs[MB];
            const uint8_t *const xsl = sc + (TN + wm * MB * 32 + l32) * BPS + kq * (BPS / 2);
#pragma unroll
            for (int b = 0; b < MB; ++b) xs[b] = BPS == 8 ? *reinterpret_cast<const uint32_t *>(xsl + b * 32 * BPS) : *reinterpret_cast<const uint16_t *>(xsl + b * 32 * BPS);
            auto slice = [&](auto jc) {
                constexpr int j = decltype(jc)::value;
                i32x8 w[NB], x[MB];
#pragma unroll
                for (int a = 0; a < NB; ++a) w[a] = mx_operand(*reinterpret_cast<const u32x4 *>(wl + a * 32 * C::WROW + 16 * ((kq * (BPS / 2) + j) ^ wkey)));
#pragma unroll
                for (int b = 0; b < MB; ++b) x[b] = mx_operand(*reinterpret_cast<const u32x4 *>(xl + b * 32 * C::XROW + 16 * ((kq * (BPS / 2) + j) ^ xkey)));
#pragma unroll
                for (int a = 0; a < NB; ++a)
#pragma unroll
                    for (int b = 0; b < MB; ++b)
                        acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[a], x[b], acc[a][b], 4, 4, j, (int)ws[a], j, (int)xs[b]);
            };
            slice(std::integral_constant<int, 0>{});
            slice(std::integral_constant<int, 1>{});
            if constexpr (BPS == 8) {
                slice(std::integral_constant<int, 2>{});
                slice(std::integral_constant<int, 3>{});
            }
        } else {
#pragma unroll
            for (int h = 0; h < BPS / 2; ++h) {  // the lane's blocks: kq * BPS / 2 + h
                u32x4 q[NB];
                float s[NB];
                const int blk = kq * (BPS / 2) + h;
#pragma unroll
                for (int a = 0; a < NB; ++a) {
                    q[a] = *reinterpret_cast<const u32x4 *>(wl + a * 32 * C::WROW + 16 * (blk ^ wkey));
                    s[a] = mx_scale((ws[a] >> (8 * h)) & 255u);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int piece = blk * 4 + j;  // of 8 bf16
                    bf16x8 x[MB];
#pragma unroll
                    for (int b = 0; b < MB; ++b)
                        x[b] = *reinterpret_cast<const bf16x8 *>(xl + piece / 8 * (TM * 128) + b * 4096 + 16 * ((piece % 8) ^ xkey));
#pragma unroll
                    for (int a = 0; a < NB; ++a) {
                        const bf16x8 w = dequant8_mx(q[a][j], s[a]);
#pragma unroll
                        for (int b = 0; b < MB; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(w, x[b], acc[a][b], 0, 0, 0);
                    }
                }
            }
        }
        keep(i + 1);
        slot = slot + 1 == ST ? 0 : slot + 1;
    }

    wait_vmcnt<0>();  // (the last requests, of zeros that nobody reads: no memory of this workgroup may be written once it has ended)
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
        float *const y = reinterpret_cast<float *>(p.y);
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

template <bool X4, bool GATED, int WN, int WM, int NB, int MB, int BPS, int ST>
static int launch(const MxProduct &p, hipStream_t st) {
    typedef Cfg<X4, WN, WM, NB, MB, BPS, ST> C;
    constexpr int TO = GATED ? C::TN / 2 : C::TN, LDS = C::lds(TO);
    static_assert(LDS <= 163840, "LDS of a compute unit");
    const int64_t tm = p.offsets ? mx_most_tiles(p.M, p.E, C::TM) : (p.M + C::TM - 1) / C::TM, tiles = tm * ((p.N + TO - 1) / TO);
    if (tiles > INT32_MAX - 8) return fail(CHADQ_ERR_SHAPE, "mxfp4 product: M=%d N=%d are too many tiles", p.M, p.N);
    static std::atomic<bool> set[64];  // more LDS than the default limit: once per device
    int dev = 0;
    CHADQ_HIP(hipGetDevice(&dev));
    if (dev >= 64 || !set[dev].load()) {
        CHADQ_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(&mx_tile_kernel<X4, GATED, WN, WM, NB, MB, BPS, ST>), hipFuncAttributeMaxDynamicSharedMemorySize, LDS));
        if (dev < 64) set[dev].store(true);
    }
    hipLaunchKernelGGL((mx_tile_kernel<X4, GATED, WN, WM, NB, MB, BPS, ST>), dim3((int)((tiles + 7) / 8 * 8)), dim3(C::T), LDS, st, p);
    return hip_check(hipGetLastError(), "mxfp4 product launch");
}

}  // namespace mxt

// The requests' offsets are 32-bit, up to 256 rows from a tile's first, or (rows read through an index) from x's first.
bool mx_tile_ok(const MxProduct &p) {
    const int64_t row = p.xs ? p.K / 2 : (int64_t)p.K * 2;
    return row * 256 < INT32_MAX && (!p.rows || row * p.x_rows < INT32_MAX);
}

int mx_tile_launch(const MxProduct &p, hipStream_t st) {
    using namespace mxt;
    if (p.w2) return launch<false, true, 2, 4, 2, 1, 4, 3>(p, st);  // 128 weight rows (64 results) x 128
    if (p.xs) return launch<true, false, 2, 4, 4, 2, 4, 4>(p, st);  // 256 x 256
    return launch<false, false, 4, 2, 1, 2, 4, 3>(p, st);           // 128 x 128
}

}  // namespace chadq
