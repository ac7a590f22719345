// Products on FP8 weights: which kernel, which tile, K in how many parts.
#include <cmath>

#include "fp8.h"

namespace chadq {

// Time of a product by tile: `start` us once, and for each round of the compute units' workgroups `round` us and `few` (64 workgroups, at the clock that they leave) to
// `full` (256) us per 1024 k.
struct TileTime {
    int tn, tm;
    float start, round, few, full;
};
static const TileTime kBf16[F8_TILES] = {{64, 32, 1.43f, 3.38f, 1.77f, 2.51f}, {64, 64, 1.25f, 4.1f, 2.46f, 3.5f}, {128, 64, 1.15f, 3.7f, 3.87f, 5.58f}, {256, 64, 0.92f, 5.05f, 6.43f, 9.74f},
                                         {128, 128, 0.57f, 5.56f, 6.05f, 8.52f}, {256, 128, 0.5f, 5.73f, 10.42f, 15.42f}, {256, 256, 0.f, 1e9f, 0.f, 0.f}};
static const TileTime kFp8[F8_TILES] = {{64, 32, 1.29f, 3.91f, 1.26f, 1.49f}, {64, 64, 0.87f, 4.66f, 1.93f, 2.4f}, {128, 64, 0.78f, 4.51f, 2.83f, 3.46f}, {256, 64, 1.04f, 3.74f, 5.09f, 6.73f},
                                        {128, 128, 0.44f, 5.13f, 4.24f, 5.92f}, {256, 128, 0.0f, 5.59f, 6.56f, 9.49f}, {256, 256, 0.43f, 6.25f, 10.36f, 19.67f}};

static Fp8TilePick pick(int M, int N, int K, int E, bool x_fp8, bool gated, int most_parts) {
    Fp8TilePick best = {F8_128x128, 0};
    float least = 1e30f;
    for (int i = 0; i < F8_TILES; ++i) {
        const TileTime &t = (x_fp8 ? kFp8 : kBf16)[i];
        const int tn = gated ? t.tn / 2 : t.tn;
        if (t.round > 1e8f || (gated && (t.tn < 128 || i == F8_128x128 || i == F8_256x256))) continue;
        // rows by group: between the tiles of groups of one size and those of exponentially distributed sizes
        const float mean = (float)M / E > 1.f ? (float)M / E : 1.f, hit = E * (1.f - expf(-(float)M / E)), even = mean / t.tm + 0.3f;
        const float tm = E > 1 ? hit * 0.5f * ((even > 1.f ? even : 1.f) + 1.f / (1.f - expf(-t.tm / mean))) : (float)mx_ceil(M, t.tm);
        const float tiles = tm * mx_ceil(N, tn);
        for (int parts = 1; parts <= most_parts; ++parts) {
            const int part_k = parts > 1 ? ((K + parts - 1) / parts + 1023) / 1024 * 1024 : K;
            if (parts > 1 && (int64_t)part_k * (parts - 1) >= K) continue;
            const float wgs = tiles * parts, full = wgs >= 256.f ? 1.f : wgs <= 64.f ? 0.f : (wgs - 64.f) / 192.f;
            // (by group: a workgroup finds its tile first; the groups' tiles end unevenly)
            const float rounds = E > 1 && wgs > 256.f ? wgs / 256.f + 0.6f : ceilf(wgs / 256.f), round = E > 1 ? t.round + 2.f : t.round;
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
    return pick(p.M, p.N, p.K, p.offsets ? p.E : 1, p.xs != nullptr, p.w2 != nullptr, most_parts);
}

int fp8_product_part_k(const Fp8Product &p, int most_parts) { return fp8_streams(p) || !fp8_tile_ok(p) ? 0 : fp8_tile_pick(p, most_parts).part_k; }

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
    if (fp8_streams(p) || !fp8_tile_ok(p)) return fp8_stream_launch(p, st);
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
