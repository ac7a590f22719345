// Products on FP8 weights: which kernel, which tile, K in how many parts.
#include <cmath>

#include "fp8.h"

namespace chadq {

// Time of a product by tile: `start` us once, and for each round of the compute units' workgroups (`wgs` to each) `round` us and `few` (a quarter of that many, at the clock
// that they leave) to `full` us per 1024 k.  Fitted to the times of every tile.
struct TileTime {
    int tn, tm, wgs;
    float start, round, few, full;
};
static const TileTime kBf16[F8_TILES] = {{64, 32, 1, 1.44f, 3.34f, 1.8f, 2.53f}, {64, 64, 1, 1.21f, 4.03f, 2.49f, 3.58f}, {128, 64, 1, 1.14f, 3.66f, 3.9f, 5.55f}, {128, 64, 2, 1.5f, 2.95f, 5.72f, 10.44f},
                                         {256, 64, 1, 0.73f, 4.98f, 6.76f, 9.67f}, {256, 64, 2, 2.29f, 2.78f, 8.27f, 20.63f}, {128, 128, 1, 0.63f, 5.37f, 6.14f, 8.53f}, {128, 128, 2, 2.15f, 2.96f, 8.34f, 19.24f},
                                         {256, 128, 1, 0.13f, 5.91f, 10.51f, 15.82f}, {256, 256, 1, 0.0f, 1e9f, 0.0f, 0.0f}};
static const TileTime kFp8[F8_TILES] = {{64, 32, 1, 1.49f, 3.78f, 1.19f, 1.49f}, {64, 64, 1, 1.28f, 4.48f, 1.77f, 2.35f}, {128, 64, 1, 0.69f, 4.73f, 2.77f, 3.42f}, {128, 64, 2, 0.47f, 3.99f, 3.46f, 6.55f},
                                        {256, 64, 1, 0.01f, 4.83f, 5.1f, 6.36f}, {256, 64, 2, 0.0f, 1e9f, 0.0f, 0.0f}, {128, 128, 1, 0.0f, 5.67f, 4.2f, 5.59f}, {128, 128, 2, 0.0f, 4.46f, 5.46f, 10.58f},
                                        {256, 128, 1, 0.0f, 5.74f, 6.48f, 9.41f}, {256, 256, 1, 0.0f, 6.9f, 10.4f, 18.19f}};
static Fp8TilePick pick(int M, int N, int K, int E, bool x_fp8, bool gated, bool h8, int most_parts) {
    Fp8TilePick best = {F8_128x128, 0};
    float least = 1e30f;
    for (int i = 0; i < F8_TILES; ++i) {
        const TileTime &t = (x_fp8 ? kFp8 : kBf16)[i];
        const int tn = gated ? t.tn / 2 : t.tn;
        if (t.round > 1e8f || (gated && (t.tn < 128 || i == F8_128x128 || i == F8_256x256 || (h8 && t.tn < 256)))) continue;
        // rows by group: between the tiles of groups of one size and those of exponentially distributed sizes
        const float mean = (float)M / E > 1.f ? (float)M / E : 1.f, hit = E * (1.f - expf(-(float)M / E)), even = mean / t.tm + 0.3f;
        const float tm = E > 1 ? hit * 0.5f * ((even > 1.f ? even : 1.f) + 1.f / (1.f - expf(-t.tm / mean))) : (float)mx_ceil(M, t.tm);
        const float tiles = tm * mx_ceil(N, tn);
        for (int parts = 1; parts <= most_parts; ++parts) {
            const int part_k = parts > 1 ? ((K + parts - 1) / parts + 1023) / 1024 * 1024 : K;
            if (parts > 1 && (int64_t)part_k * (parts - 1) >= K) continue;
            const float at_once = 256.f * t.wgs, w = tiles * parts / at_once, full = w >= 1.f ? 1.f : w <= 0.25f ? 0.f : (w - 0.25f) / 0.75f;
            // (by group: a workgroup finds its tile first; the groups' tiles end unevenly)
            const float rounds = E > 1 && w > 1.f ? w + 0.6f : ceilf(w), round = E > 1 ? t.round + 2.f : t.round;
            float us = t.start + rounds * (round + (t.few + (t.full - t.few) * full) * (part_k / 1024.f));
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
    return pick(p.M, p.N, p.K, p.offsets ? p.E : 1, p.xs != nullptr, p.w2 != nullptr, p.h8 != nullptr, most_parts);
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
