// Microscaled 4-bit floating point (MXFP4): what its kernels share.
//   codes  e2m1: sign in bit 3, then 0, 0.5, 1, 1.5, 2, 3, 4, 6; two to a byte, even k in the low nibble
//   scales e8m0: one byte e per 32 codes along K, 2^(e - 127); 255: the block is NaN
// The conversions of this machine read the exponent field of a scale given as a float: e << 23 serves for every byte (0 reads
// as 2^-127, 255 as NaN; all 256 bytes x 16 codes checked).
#pragma once
#include <type_traits>

#include "chadq_common.h"

namespace chadq {

typedef __attribute__((ext_vector_type(8))) int32_t i32x8;

__device__ __forceinline__ float mx_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// 8 codes (one word) -> 8 bf16 in k order, times the block's scale: exact, one instruction per pair
__device__ __forceinline__ bf16x8 dequant8_mx(uint32_t w, float s) {
    const u32x4 r = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3))};
    bf16x8 o;
    __builtin_memcpy(&o, &r, 16);
    return o;
}

// The bare barrier behind a wait for the wave's own LDS accesses (__syncthreads() would also wait for every outstanding memory request); the
// empty asm statements keep the compiler from moving LDS accesses across it.
__device__ __forceinline__ void wg_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A value that is the same in every lane, for the compiler: a buffer's descriptor from a pointer that it takes for a lane's own costs a loop per request.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint8_t *uniform(const void *p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<uint8_t *>((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}

// 32 codes as the operand of a scaled MFMA (fp4 takes the lower half of its eight registers)
__device__ __forceinline__ i32x8 mx_operand(u32x4 v) {
    const auto w = __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1);
    return __builtin_bit_cast(i32x8, w);
}

// B scale bytes (1, 2, 4 or 8, no more than the row has) from byte `at` of a row of G on, zeros behind its end (2^-127: what is infinite may not
// meet the activations there, which are zeros); any alignment.  What is loaded near the end begins before `at`: the shift that puts that right is left
// to the reader (get), who does not want to wait for it earlier.
template <int B>
struct MxScales {
    typedef std::conditional_t<B == 8, uint64_t, std::conditional_t<B == 4, uint32_t, std::conditional_t<B == 2, uint16_t, uint8_t>>> bytes_t;
    bytes_t raw;
    int cut;
    __device__ __forceinline__ void load(const uint8_t *row, int at, int G) {
        const int o = at < G - B ? at : G - B;
        cut = at - o < B ? at - o : B;
        __builtin_memcpy(&raw, row + o, B);
    }
    __device__ __forceinline__ bytes_t get() const { return cut < B ? (bytes_t)(raw >> (8 * cut)) : (bytes_t)0; }
};

// y[r, n] = sum_k x[r, k] w[g(r), n, k] for the rows r of group g(r) = the g with offsets[g] <= r < offsets[g + 1]
struct MxProduct {
    const void *x;            // bf16 [M,K], or codes [M,K/2]
    const uint8_t *xs;        // scales of the codes [M,K/32]
    const uint8_t *w, *ws;    // codes [E,N,K/2], scales [E,N,K/32]
    void *y;                  // fp32 or bf16 [M,N]
    const int32_t *offsets;   // [E+1] on the device, or null: one group, all rows
    int M, N, K, E;
    bool y_bf16, clear_rest;  // clear_rest: rows of no group become 0 (else they are left as they are)
    // mixture of experts: row r of the groups is row rows[r] of x (null: r); with a second matrix per group, of w's shape, the result
    // is bf16( silu(x w) (x w2) )
    const int32_t *rows = nullptr;
    int x_rows = 0;           // ... which has so many
    const uint8_t *w2 = nullptr, *w2s = nullptr;
    // K in parts of part_k (a multiple of 512; 0: one part), the sums of part i as fp32 [M,N] from y + i M N on
    int part_k = 0;
    int parts() const { return part_k ? (K + part_k - 1) / part_k : 1; }
};

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.f + __expf(-g)) * u; }

// Row tiles of the groups, TR rows to a tile, a group's last one cut; behind them the tiles of the rows of no group (in front of offsets[0] and
// behind offsets[E]), for those who clear them.  Offsets are taken as clamped into [0, M] and never descending (one that descends counts as
// the largest before it), so that no contents of theirs lead outside x and y.  Every lane of a wave calls this; the answers are uniform.
struct MxTile {
    int group, row0, rows, rest0, rest1;  // group -1: rows of no group, counted as rest0 rows from 0 on and then the rows from rest1 on
};
// Inclusive scan over the wave's lanes, of values that are not negative: inside the 16-lane rows, then across them
template <typename OP>
__device__ __forceinline__ int wave_scan(int v, OP op) {
#define CHADQ_SCAN_STEP(CTRL, MASK) v = op(v, __builtin_amdgcn_update_dpp(0, v, CTRL, MASK, 0xF, false));
    CHADQ_SCAN_STEP(0x111, 0xF)  // row_shr 1, 2, 4, 8
    CHADQ_SCAN_STEP(0x112, 0xF)
    CHADQ_SCAN_STEP(0x114, 0xF)
    CHADQ_SCAN_STEP(0x118, 0xF)
    CHADQ_SCAN_STEP(0x142, 0xA)  // row_bcast15 into rows 1 and 3
    CHADQ_SCAN_STEP(0x143, 0xC)  // row_bcast31 into rows 2 and 3
#undef CHADQ_SCAN_STEP
    return v;
}

struct MxTiles {
    const int32_t *__restrict__ offsets;
    int E, M, TR;

    // 64 groups from c on: the lane's first row, the one behind its last, and tiles up to and with it; low: largest offset so far
    __device__ __forceinline__ void scan(int c, int low, int &lo, int &hi, int &upto) const {
        const int lane = threadIdx.x & 63, e = c + lane;
        auto at = [&](int i) {
            const int o = offsets[i < E ? i : E];
            return o < 0 ? 0 : o > M ? M : o;
        };
        lo = at(e);
        const int next = at(e + 1);
        lo = wave_scan(lo > low ? lo : low, [](int a, int b) { return a > b ? a : b; });
        hi = next > lo ? next : lo;
        upto = wave_scan(e < E ? (hi - lo + TR - 1) / TR : 0, [](int a, int b) { return a + b; });
    }
    // Tiles of the groups, and (clear) of the rows of none.  at(tiles): which tile the workgroup takes of so many (or -1: none).  Returns that tile.
    // One pass over the offsets where they are few, as their round trip to memory is what a workgroup begins with.
    template <typename F>
    __device__ __forceinline__ MxTile place(bool clear, F at) const {
        int before = 0, low = 0, first = 0, lo, hi, upto;
        for (int c = 0; c < E; c += 64) {
            scan(c, low, lo, hi, upto);
            if (c == 0) first = __builtin_amdgcn_readlane(lo, 0);
            before += __builtin_amdgcn_readlane(upto, 63);
            low = __builtin_amdgcn_readlane(hi, 63);
        }
        const int rest = first + (M - low), t = at(before + (clear ? (rest + TR - 1) / TR : 0));
        if (t < 0) return {-1, 0, 0, 0, 0};
        if (t >= before) {
            const int r0 = (t - before) * TR;
            return {-1, r0, rest - r0 < 0 ? 0 : rest - r0 < TR ? rest - r0 : TR, first, low};
        }
        before = low = 0;
        for (int c = 0; c < E; c += 64) {
            if (E > 64) scan(c, low, lo, hi, upto);
            const unsigned long long m = __ballot(t < before + upto);
            if (m) {
                const int l = __ffsll((long long)m) - 1, r0 = __builtin_amdgcn_readlane(lo, l), end = __builtin_amdgcn_readlane(hi, l);
                const int r = r0 + (t - before - (__builtin_amdgcn_readlane(upto, l) - (end - r0 + TR - 1) / TR)) * TR;
                return {c + l, r, end - r < TR ? end - r : TR, 0, 0};
            }
            before += __builtin_amdgcn_readlane(upto, 63);
            low = __builtin_amdgcn_readlane(hi, 63);
        }
        return {-1, 0, 0, 0, 0};
    }
    __device__ __forceinline__ MxTile find(int t) const {
        return place(false, [t](int) { return t; });
    }
};
// a / b rounded up; rows and columns up to 2^31 - 1 with a tile more do not fit 32 bits
inline int64_t mx_ceil(int64_t a, int64_t b) { return (a + b - 1) / b; }
// Row tiles that suffice for any offsets: full tiles of M rows, one cut per group that can have a row, one of the rest.
inline int64_t mx_most_tiles(int M, int E, int TR) { return (int64_t)M / TR + (E < M ? E : M) + 2; }

// The columns n0 .. n0 + cols of the tile's rows of no group, set to 0 by the workgroup's threads
__device__ __forceinline__ void mx_clear(void *y, bool y_bf16, int N, const MxTile &t, int n0, int cols) {
    const int width = N - n0 < cols ? N - n0 : cols;
    for (int i = threadIdx.x; i < t.rows * width; i += blockDim.x) {
        const int k = t.row0 + i / width, r = k < t.rest0 ? k : t.rest1 + (k - t.rest0);
        store_sum(reinterpret_cast<float *>(y), (size_t)r * N + n0 + i % width, 0.f, y_bf16);
    }
}

bool mx_streams(const MxProduct &p);
int mx_stream_launch(const MxProduct &p, hipStream_t st);
bool mx_tile_ok(const MxProduct &p);
struct MxTilePick {
    int tile, part_k;  // 0: one part
};
constexpr int kMxMostK = 1 << 26;  // bytes of an activation row are counted in 32 bits
constexpr int kMxParts = 8, kMxGroupParts = 4;  // parts of K at most, of a product by group (which its caller joins)
MxTilePick mx_tile_pick(const MxProduct &p, int most_parts);
int mx_tile_launch(const MxProduct &p, int tile, hipStream_t st);
int mx_tile_parts_launch(const MxProduct &p, int tile, float *part, hipStream_t st);
int mx_join_launch(const float *part, void *y, int64_t n, int parts, bool y_bf16, hipStream_t st);
int mx_product_part_k(const MxProduct &p, int most_parts);
int mx_product_launch(const MxProduct &p, void *workspace, size_t workspace_bytes, hipStream_t st);
size_t mx_product_workspace_bytes(int M, int N, int K, bool x_mxfp4);

}  // namespace chadq
