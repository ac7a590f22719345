// Products on FP8 weights: which kernel, which tile, K in how many parts.
#include <cmath>

#include "fp8.h"

namespace chadq {

// Time of a product by tile: `start` us once, and for each round of the compute units' workgroups (`wgs` to each) `round` us and `few` (a quarter of that many, at the clock
// that they leave) to `full` us per 1024 k.  Fitted to the times of every tile in 1400 products with random sizes (17 to 8192 rows, 64 to 14336 columns, k of 128 to 14336,
// up to 64 groups).  On 240 others the tile taken is on average 2 to 4 % slower than the fastest of all tiles and parts.
struct TileTime {
    int tn, tm, wgs;
    float start, round, few, full;
    float per_k(float share) const { return few + (full - few) * (share >= 1.f ? 1.f : share <= 0.25f ? 0.f : (share - 0.25f) / 0.75f); }
};
static const TileTime kBf16[F8_TILES] = {{64, 32, 1, 2.28f, 2.1f, 1.87f, 2.73f}, {64, 64, 1, 2.29f, 2.48f, 2.52f, 3.57f}, {128, 64, 1, 1.93f, 2.36f, 4.07f, 6.1f}, {128, 64, 2, 2.32f, 1.55f, 5.98f, 12.33f},
                                         {256, 64, 1, 1.5f, 3.62f, 6.95f, 11.16f}, {256, 64, 2, 2.13f, 2.22f, 9.05f, 23.11f}, {128, 128, 1, 1.62f, 3.87f, 6.58f, 8.75f}, {128, 128, 2, 2.42f, 2.31f, 8.56f, 17.26f},
                                         {256, 128, 1, 1.26f, 4.33f, 10.91f, 16.05f}, {256, 256, 1, 0.0f, 1e9f, 0.0f, 0.0f}};
static const TileTime kFp8[F8_TILES] = {{64, 32, 1, 2.13f, 2.47f, 1.18f, 1.86f}, {64, 64, 1, 2.41f, 2.64f, 1.7f, 2.86f}, {128, 64, 1, 2.14f, 2.38f, 2.61f, 4.48f}, {128, 64, 2, 2.16f, 1.72f, 3.62f, 8.51f},
                                        {256, 64, 1, 1.28f, 2.86f, 4.85f, 8.03f}, {256, 64, 2, 0.0f, 1e9f, 0.0f, 0.0f}, {128, 128, 1, 2.24f, 2.79f, 4.06f, 6.65f}, {128, 128, 2, 2.26f, 1.63f, 5.19f, 12.67f},
                                        {256, 128, 1, 1.11f, 3.87f, 6.66f, 10.62f}, {256, 256, 1, 2.73f, 3.14f, 10.74f, 16.61f}};
static Fp8TilePick pick(int M, int N, int K, int E, bool x_fp8, bool gated, int most_parts) {
    Fp8TilePick best = {F8_128x128, 0};
    float least = 1e30f;
    for (int i = 0; i < F8_TILES; ++i) {
        const TileTime &t = (x_fp8 ? kFp8 : kBf16)[i];
        const int tn = gated ? t.tn / 2 : t.tn;
        // (gate and up: half the columns of each; results of 8 bits need a whole block of 128)
        if (t.round > 1e8f || (gated && (t.tn < (x_fp8 ? 256 : 128) || i == F8_128x128 || i == F8_256x256))) continue;
        // rows by group: between the tiles of groups of one size and those of exponentially distributed sizes
        const float mean = (float)M / E > 1.f ? (float)M / E : 1.f, hit = E * (1.f - expf(-(float)M / E)), even = mean / t.tm + 0.3f;
        const float tm = E > 1 ? hit * 0.5f * ((even > 1.f ? even : 1.f) + 1.f / (1.f - expf(-t.tm / mean))) : (float)mx_ceil(M, t.tm);
        const float tiles = tm * mx_ceil(N, tn);
        for (int parts = 1; parts <= most_parts; ++parts) {
            const int part_k = parts > 1 ? ((K + parts - 1) / parts + 1023) / 1024 * 1024 : K;
            if (parts > 1 && (int64_t)part_k * (parts - 1) >= K) continue;
            const float w = tiles * parts / (256.f * t.wgs), chunks = part_k / 1024.f;
            float us;
            if (E > 1) {  // a workgroup finds its tile first; the groups' tiles end unevenly
                us = t.start + (w > 1.f ? w + 0.6f : 1.f) * (t.round + 2.f + t.per_k(w) * chunks);
            } else {
                const float whole = floorf(w), rest = w - whole;
                us = t.start + whole * (t.round + t.full * chunks) + (rest > 0.f ? t.round + t.per_k(rest) * chunks : 0.f);
            }
            if (parts > 1) us += 3.f + (8.f * parts + 2.f) * M * (float)N * 2.5e-7f;  // the sums written, read again and joined by another launch
            if (us < least * (parts > 1 ? 0.95f : 1.f)) {
                least = us;
                best = {i, parts > 1 ? part_k : 0};
            }
        }
    }
    return best;
}

Fp8TilePick fp8_tile_pick(const Fp8Product &p, int most_parts) {
    return pick(p.M, p.N, p.K, p.offsets ? p.E : 1, p.xs != nullptr, p.w2 != nullptr, most_parts);
}

// Which of the two: the tiles' requests do not reach over rows as long as the streams' do
bool fp8_product_streams(const Fp8Product &p) { return fp8_streams(p) || !fp8_tile_ok(p); }

int fp8_product_part_k(const Fp8Product &p, int most_parts) { return fp8_product_streams(p) ? 0 : fp8_tile_pick(p, most_parts).part_k; }

size_t fp8_product_workspace_bytes(int M, int N, int K, bool x_fp8) {
    Fp8Product p = {};
    p.M = M;
    p.N = N;
    p.K = K;
    p.E = 1;
    static const float any = 0.f;
    p.xs = x_fp8 ? &any : nullptr;
    p.part_k = fp8_product_part_k(p, kFp8Parts);
    return p.part_k ? (size_t)p.parts() * M * N * 4 : 0;
}

int fp8_product_launch(const Fp8Product &p, void *workspace, size_t workspace_bytes, hipStream_t st) {
    if (fp8_product_streams(p)) return fp8_stream_launch(p, st);
    if (p.part_k) return fp8_tile_launch(p, fp8_tile_pick(p, kFp8GroupParts).tile, st);  // (the caller, who asked for at most so many, joins the parts)
    if (!p.offsets && workspace) {
        Fp8Product q = p;
        const Fp8TilePick pick = fp8_tile_pick(p, kFp8Parts);
        q.part_k = pick.part_k;
        if (pick.part_k && workspace_bytes >= (size_t)q.parts() * p.M * p.N * 4) {
            q.y = workspace;
            q.y_bf16 = false;
            const int rc = fp8_tile_launch(q, pick.tile, st);
            return rc ? rc : mx_join_launch(reinterpret_cast<const float *>(workspace), p.y, (int64_t)p.M * p.N, q.parts(), p.y_bf16, st);
        }
    }
    return fp8_tile_launch(p, fp8_tile_pick(p, 1).tile, st);
}

}  // namespace chadq
