// Routing to up to 512 experts, and the sorting of the chosen pairs by expert.
#pragma once
#include "chadq_common.h"

namespace chadq {

constexpr int kRouteExperts = 512, kRouteTopK = 32, kRouteGroups = 64;
constexpr int kSortChunk = 1024, kSortAlone = 12;  // pairs to a workgroup; workgroups up to which each counts all pairs

struct Routing {
    const float *bias;  // [E] or null
    int sigmoid, renorm, groups, top_groups, group_sum, top_k;
    float scale;
};
// Pairs p = t * top_k + slot by expert, the order of p kept inside an expert
struct RouteSort {
    int32_t *pos;      // [P] row of the pair
    int32_t *tok;      // [P] token of the row
    int32_t *offsets;  // [E+1] first row of each expert
    int32_t *hist;     // [chunks,E], for more than kSortAlone chunks
};
inline int sort_chunks(int64_t P) { return (int)((P + kSortChunk - 1) / kSortChunk); }

int route_experts_launch(const float *logits, int32_t *idx, float *w, int T, int E, const Routing &r, hipStream_t st);
// the same, and the pairs sorted
int route_sort_launch(const float *logits, int32_t *idx, float *w, int T, int E, const Routing &r, const RouteSort &s, hipStream_t st);

}  // namespace chadq
