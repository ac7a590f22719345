// 8-bit floating point (FP8) with a scale for each block of 128: what its kernels share.
//   values e4m3: sign, 4 bits of exponent (bias 7), 3 of mantissa; largest 448, 0x7F and 0xFF are NaN; one to a byte
//   scales fp32: of activations one per row and 128 k, of weights one per 128 rows and 128 k; the last block of rows and of k may be cut
// A product's sum of a block, of values alone, is multiplied by the block's scales and added to the result, all in fp32.
#pragma once
#include "mx.h"

namespace chadq {

constexpr int kFp8Block = 128;
inline __host__ __device__ int fp8_blocks(int n) { return (int)(((int64_t)n + 127) >> 7); }

// 4 values (one word) -> 4 bf16 in order, exact
__device__ __forceinline__ u32x2 fp8_to_bf16(uint32_t w) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true))};
}

// Quantisation of a block with a = max(max |x|, 448 * 2^-126):
//   scale = a / 448,  r = 448 / a  (fp32 divisions),  value = the nearest e4m3 to x r (one fp32 product), ties to the even one.
// |x r| <= 448 (1 + 2^-23), which goes to 448: nothing saturates.  The least a keeps scale and r normal numbers.  A block that holds a NaN or an
// infinity gets a NaN for its scale and values of 0.
constexpr float kFp8Least = 448.f * 0x1p-126f;

__device__ __forceinline__ uint32_t absmax8(const float f[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t b = __float_as_uint(f[j]) & 0x7FFFFFFFu;  // as integers: a NaN is larger than infinity
        m = b > m ? b : m;
    }
    return m;
}

struct Fp8Scale {
    float scale, r;
    bool bad;
    __device__ __forceinline__ explicit Fp8Scale(uint32_t most) {
        bad = most >= 0x7F800000u;
        const float m = __uint_as_float(most), a = m > kFp8Least ? m : kFp8Least;
        scale = bad ? __uint_as_float(0x7FC00000u) : a / 448.f;
        r = 448.f / a;
    }
    __device__ __forceinline__ u32x2 values(const float f[8]) const {
        int lo = 0, hi = 0;
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] * r, f[1] * r, lo, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2] * r, f[3] * r, lo, true);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4] * r, f[5] * r, hi, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6] * r, f[7] * r, hi, true);
        return bad ? u32x2{0, 0} : u32x2{(uint32_t)lo, (uint32_t)hi};
    }
};

// over 16 lanes next to each other
__device__ __forceinline__ uint32_t max_of_16(uint32_t m) {
#define CHADQ_MAX_STEP(CTRL)                                                                                \
    {                                                                                                       \
        const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, CTRL, 0xF, 0xF, false);         \
        m = o > m ? o : m;                                                                                  \
    }
    CHADQ_MAX_STEP(0xB1)   // quad_perm [1,0,3,2]
    CHADQ_MAX_STEP(0x4E)   // quad_perm [2,3,0,1]
    CHADQ_MAX_STEP(0x141)  // row_half_mirror
    CHADQ_MAX_STEP(0x140)  // row_mirror
#undef CHADQ_MAX_STEP
    return m;
}

// y[r, n] = sum over blocks b of xs[r, b] ws[g(r), n / 128, b] sum_{k in b} x[r, k] w[g(r), n, k] for the rows r of group g(r) = the g with
// offsets[g] <= r < offsets[g + 1]
struct Fp8Product {
    const void *x;            // bf16 [M,K] (xs null), or values [M,K]
    const float *xs;          // scales of the values [M,ceil(K/128)]
    const uint8_t *w;         // values [E,N,K]
    const float *ws;          // [E,ceil(N/128),ceil(K/128)]
    void *y;                  // fp32 or bf16 [M,N]
    const int32_t *offsets;   // [E+1] on the device, or null: one group, all rows
    int M, N, K, E;
    bool y_bf16, clear_rest;  // clear_rest: rows of no group become 0 (else they are left as they are)
    // mixture of experts: row r of the groups is row rows[r] of x (null: r); with a second matrix per group, of w's shape, the result
    // is silu(x w) (x w2)
    const int32_t *rows = nullptr;
    int x_rows = 0;           // ... which has so many
    const uint8_t *w2 = nullptr;
    const float *w2s = nullptr;
    // ... with 8-bit x and more rows than are streamed always in 8 bits: values [M,N], scales [M,ceil(N/128)] (then y is not written)
    uint8_t *h8 = nullptr;
    float *h8s = nullptr;
    // K in parts of part_k (a multiple of 1024; 0: one part), the sums of part i as fp32 [M,N] from y + i M N on
    int part_k = 0;
    int parts() const { return part_k ? (K + part_k - 1) / part_k : 1; }
};

constexpr int kFp8MostK = 1 << 26;  // bytes of an activation row are counted in 32 bits

// weight rows x activation rows; P: two workgroups to a compute unit
enum Fp8Tile { F8_64x32, F8_64x64, F8_128x64, F8_128x64P, F8_256x64, F8_256x64P, F8_128x128, F8_128x128P, F8_256x128, F8_256x256, F8_TILES };
struct Fp8TilePick {
    int tile, part_k;  // 0: one part
};
constexpr int kFp8Parts = 8, kFp8GroupParts = 4;  // parts of K at most, of a product by group (which its caller joins)
bool fp8_streams(const Fp8Product &p);
int fp8_stream_launch(const Fp8Product &p, hipStream_t st);
bool fp8_product_streams(const Fp8Product &p);
bool fp8_tile_ok(const Fp8Product &p);
Fp8TilePick fp8_tile_pick(const Fp8Product &p, int most_parts);
int fp8_tile_launch(const Fp8Product &p, int tile, hipStream_t st);
int fp8_product_part_k(const Fp8Product &p, int most_parts);
int fp8_product_launch(const Fp8Product &p, void *workspace, size_t workspace_bytes, hipStream_t st);
size_t fp8_product_workspace_bytes(int M, int N, int K, bool x_fp8);

}  // namespace chadq
