// Routing to experts.  Token t with logits z over E experts in `groups` groups of consecutive ones:
//   score s = softmax(z) or 1 / (1 + exp(-z));  an expert is chosen by c = s + bias, or by z where there is neither a bias nor a sum over a group
//   a group's value is the sum of its group_sum largest c; the experts of the top_groups largest groups are open
//   the top_k open experts with the largest c, ties to the lowest index;  weights s, divided by their sum if asked (0 where that is 0), times scale
// An expert whose logit is -infinity or NaN (a masked one) comes behind all others that are open, also behind those that a bias of -infinity switches off, and has
// the score 0; a group with fewer than group_sum unmasked experts comes behind those that have them.  So choices are compared by keys, where a masked expert has one
// below that of -infinity.  A c that is NaN (a NaN in bias) counts as -infinity, a group's +infinity + -infinity as +infinity.
//
// c and the sums of groups are formed in 64 bits: in 32 two experts whose scores differ by less than a rounding change places, which happens to a few of some
// thousand tokens, and then another expert's output is added.  By z alone, 32 bits are exact.
//
// A token takes L lanes of a wave (8 to 64), each with PER consecutive experts: a lane's best is found among its own, the token's by a reduction over the lanes,
// and the lowest lane that holds it wins, so that equal ones go to the lowest index with no index in the keys.
// Bound by the chain of a token's rounds (a reduction over 64 lanes each, in registers) and, with many tokens, by the 64-bit exponentials and comparisons: 8 of 256
// experts in 8 groups, sigmoid and bias, 16 tokens 6.0 us, 8192 tokens 19.4 (8.4 MB: 1.6 from memory).  16 lanes of 16 experts to a token took 18.7, a choice in 32 bits first, with
// 64 where it is near, 25.
#include <type_traits>

#include "route.h"

namespace chadq {

__device__ __forceinline__ uint32_t route_key(float v) { return order_key(v); }
__device__ __forceinline__ uint64_t route_key(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
    return b ^ ((b >> 63) ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ double route_value(uint64_t key) { return __builtin_bit_cast(double, key ^ ((key >> 63) ? 1ull << 63 : ~0ull)); }
constexpr uint32_t kKeyClosed = 0, kKeyMasked = 1;  // (-infinity's, the least of a number, is larger)

// f(v, the value of the lane that differs in one bit of its number) for a value that is the same in all lanes with the same number without the lower bits
template <int S, typename T, typename F>
__device__ __forceinline__ T across(T v, F f) {
    static_assert(sizeof(T) == 4 || sizeof(T) == 8, "one or two registers");
    constexpr int N = sizeof(T) / 4;
    struct words_t { uint32_t w[N]; };
    words_t a = __builtin_bit_cast(words_t, v), b = a;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (S < 16) {  // quad_perm [1,0,3,2] and [2,3,0,1], row_half_mirror, row_mirror
            constexpr int CTRL = S == 1 ? 0xB1 : S == 2 ? 0x4E : S == 4 ? 0x141 : 0x140;
            b.w[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a.w[i], CTRL, 0xF, 0xF, false);
        } else {  // the rows, or halves, of both, one beside the other: every lane gets either
            const auto r = S == 16 ? __builtin_amdgcn_permlane16_swap(a.w[i], a.w[i], false, false) : __builtin_amdgcn_permlane32_swap(a.w[i], a.w[i], false, false);
            a.w[i] = r[0];
            b.w[i] = r[1];
        }
    }
    return f(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b));
}
// f over L lanes next to each other, the result in all of them
template <int L, typename T, typename F>
__device__ __forceinline__ T over_lanes(T v, F f) {
    if constexpr (L > 1) v = across<1>(v, f);
    if constexpr (L > 2) v = across<2>(v, f);
    if constexpr (L > 4) v = across<4>(v, f);
    if constexpr (L > 8) v = across<8>(v, f);
    if constexpr (L > 16) v = across<16>(v, f);
    if constexpr (L > 32) v = across<32>(v, f);
    return v;
}
template <int L>
__device__ __forceinline__ uint32_t most_of(uint32_t v) {
    return over_lanes<L>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
// the largest key, by its upper word and then by the lower one: a comparison of two words is no single instruction
template <int L>
__device__ __forceinline__ uint64_t most_of(uint64_t v) {
    const uint32_t hi = most_of<L>((uint32_t)(v >> 32)), lo = most_of<L>((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
    return (uint64_t)hi << 32 | lo;
}
// the value of lane `from`, one for the whole wave where a token takes all of it
template <int L, typename T>
__device__ __forceinline__ T from_lane(T v, int from) {
    if constexpr (L < 64) return __shfl(v, from);
    constexpr int N = sizeof(T) / 4;
    struct words_t { uint32_t w[N]; };
    words_t a = __builtin_bit_cast(words_t, v);
#pragma unroll
    for (int i = 0; i < N; ++i) a.w[i] = (uint32_t)__builtin_amdgcn_readlane((int)a.w[i], from);
    return __builtin_bit_cast(T, a);
}
// the two largest values of some
template <typename V>
struct Two {
    V a, b;
    __device__ __forceinline__ void take(V v) {
        b = v > a ? a : v > b ? v : b;
        a = v > a ? v : a;
    }
    template <int S>
    __device__ __forceinline__ void join() {
        const auto pick = [](V x, V y) { return x > y ? x : y; };
        // of the lane's own and the other's: the larger first, and of its loser and the seconds the largest
        V oa, ob;
        across<S>(a, [&](V x, V y) { oa = x, ob = y; return x; });
        const V first = pick(oa, ob), loser = oa > ob ? ob : oa;
        V sa, sb;
        across<S>(b, [&](V x, V y) { sa = x, sb = y; return x; });
        a = first;
        b = pick(loser, pick(sa, sb));
    }
};

// All lanes of the wave; the token's choices come back in its lanes 0 .. top_k - 1.  lds: [tokens of the workgroup][L * PER] keys (groups > 1)
template <int L, int PER, bool WIDE>
__device__ __forceinline__ void route_token_lanes(const float *__restrict__ z, int E, const Routing &r, void *lds, int &chosen, float &weight) {
    typedef std::conditional_t<WIDE, double, float> V;
    typedef std::conditional_t<WIDE, uint64_t, uint32_t> K;
    const int lane = threadIdx.x & 63, ls = lane % L, seg = lane - ls;
    const unsigned long long seg_mask = (L == 64 ? ~0ull : ((1ull << L) - 1)) << seg;
    const auto larger = [](auto a, auto b) { return a > b ? a : b; };
    float zr[PER];
    bool masked[PER];
    bool whole = false;
    if constexpr (PER % 4 == 0) {  // in quads where they are whole
        whole = E == L * PER && (reinterpret_cast<uintptr_t>(z) & 15) == 0;  // (rows of 16 bytes' multiples: all tokens alike)
        if (whole)
#pragma unroll
            for (int i = 0; i < PER / 4; ++i) {
                const f32x4 v = reinterpret_cast<const f32x4 *>(z)[ls * (PER / 4) + i];
#pragma unroll
                for (int j = 0; j < 4; ++j) zr[4 * i + j] = v[j];
            }
    }
    float bias[WIDE ? PER : 1];
    if constexpr (WIDE)
#pragma unroll
        for (int i = 0; i < PER; ++i) bias[i] = r.bias ? r.bias[ls * PER + i < E ? ls * PER + i : E - 1] : 0.f;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = ls * PER + i;
        zr[i] = whole ? zr[i] : e < E ? z[e] : -INFINITY;
        masked[i] = !(zr[i] > -INFINITY);  // NaN too
        top = masked[i] ? top : fmaxf(top, zr[i]);
    }
    top = over_lanes<L>(top, larger);
    V c[PER];      // what chooses
    V total = 0;   // of the softmax
    const float from_top = top > -INFINITY ? top : 0.f;
    if constexpr (WIDE) {
        // (one loop for each, with nothing in it to branch about: the lane's exponentials run into each other)
        if (r.sigmoid) {
#pragma unroll
            for (int i = 0; i < PER; ++i) c[i] = 1.0 / (1.0 + exp(-(double)(masked[i] ? 0.f : zr[i])));
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                c[i] = exp((double)(masked[i] ? from_top : zr[i]) - (double)from_top);
                total += masked[i] ? 0.0 : c[i];
            }
            total = over_lanes<L>(total, [](double a, double b) { return a + b; });
#pragma unroll
            for (int i = 0; i < PER; ++i) c[i] /= total;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            c[i] += (double)bias[i];
            c[i] = c[i] == c[i] ? c[i] : -INFINITY;
        }
    } else {
        if (!r.sigmoid && !r.renorm) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const float e = expf(masked[i] ? 0.f : zr[i] - from_top);
                total += masked[i] ? 0.f : e;
            }
            total = over_lanes<L>(total, [](float a, float b) { return a + b; });
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) c[i] = zr[i];
    }
    K key[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = masked[i] ? kKeyMasked : route_key(c[i]);
    uint32_t open = 0;  // bit i: expert i of the lane may still be chosen
#pragma unroll
    for (int i = 0; i < PER; ++i) open |= (ls * PER + i < E ? 1u : 0u) << i;
    if (r.groups > 1) {
        const int G = r.groups, per = E / G;
        int q;  // lanes that share a group: a power of two
        Two<K> two = {kKeyClosed, kKeyClosed};
        if (E == L * PER && per % PER == 0 && ((per / PER) & (per / PER - 1)) == 0) {  // whole lanes to a group: as they are
            q = per / PER;
#pragma unroll
            for (int i = 0; i < PER; ++i) two.take(key[i]);
        } else {  // through LDS, each of a group's lanes every q-th
            for (q = L; q * G > L;) q >>= 1;
            K *const mine = reinterpret_cast<K *>(lds) + (threadIdx.x / L) * (L * PER);
#pragma unroll
            for (int i = 0; i < PER; ++i) mine[ls * PER + i] = key[i];
            __builtin_amdgcn_wave_barrier();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // a wave's own: its LDS accesses keep their order
            if (ls / q < G)
                for (int i = ls % q; i < per; i += q) two.take(mine[ls / q * per + i]);
        }
        if (q > 1) two.template join<1>();
        if (q > 2) two.template join<2>();
        if (q > 4) two.template join<4>();
        if (q > 8) two.template join<8>();
        if (q > 16) two.template join<16>();
        const int g = ls / q;
        // (a sum of two, one of them masked: behind all sums without, by the other one)
        const bool cut = WIDE && r.group_sum == 2 && two.a > kKeyMasked && two.b <= kKeyMasked;
        K value = two.a;
        if constexpr (WIDE)
            if (r.group_sum == 2 && two.b > kKeyMasked) {
                const double sum = route_value(two.a) + route_value(two.b);
                value = sum == sum ? route_key(sum) : two.a;
            }
        const unsigned long long cuts = __ballot(cut);
        int rank = 0;
        if (!cuts) {  // (one answer for the wave)
            for (int h = 0; h < G; ++h) {
                const K o = from_lane<L>(value, seg + h * q);
                rank += o > value || (o == value && h < g);
            }
        } else {
            for (int h = 0; h < G; ++h) {
                const int from = seg + h * q;
                const K o = from_lane<L>(value, from);
                const bool ocut = cuts >> from & 1, one = ocut != cut && o > kKeyMasked && value > kKeyMasked;  // (what is all masked is behind both)
                rank += one ? cut : o > value || (o == value && h < g);
            }
        }
        const unsigned long long kept = __ballot(g < G && rank < r.top_groups) >> seg;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = ls * PER + i;
            if (e < E && !(kept >> (e / per * q) & 1)) open &= ~(1u << i);
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) key[i] = open >> i & 1 ? key[i] : kKeyClosed;
    K best;
    int at;
    auto own = [&] {
        best = key[0];
        at = 0;
#pragma unroll
        for (int i = 1; i < PER; ++i)
            if (key[i] > best) {  // strict: the lowest index
                best = key[i];
                at = i;
            }
    };
    own();
    float zc = -INFINITY;
    chosen = 0;
    for (int k = 0; k < r.top_k; ++k) {
        const K most = most_of<L>(best);
        const unsigned long long hold = __ballot(best == most) & seg_mask;
        const int winner = __ffsll((long long)hold) - 1;
        const int e = from_lane<L>(ls * PER + at, winner);
        if (ls == k) chosen = e;
        if constexpr (PER <= 4) {
            float zw = zr[0];
#pragma unroll
            for (int i = 1; i < PER; ++i) zw = at == i ? zr[i] : zw;
            zw = from_lane<L>(zw, winner);
            if (ls == k) zc = zw;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) key[i] = lane == winner && at == i ? 0 : key[i];
        own();
    }
    if constexpr (PER > 4) zc = ls < r.top_k ? z[chosen] : -INFINITY;
    // the chosen ones' scores again, from their logits
    const bool has = ls < r.top_k, none = !(zc > -INFINITY);
    const float from = !WIDE && r.renorm ? over_lanes<L>(has && !none ? zc : -INFINITY, larger) : top;
    double sc = !has || none ? 0.0 : r.sigmoid ? 1.0 / (1.0 + exp(-(double)zc)) : exp((double)zc - (double)from);
    if (!r.sigmoid && (WIDE || !r.renorm) && !none) sc /= (double)total;
    if (!has) sc = 0.0;
    if (r.renorm) {
        const double sum = over_lanes<L>(sc, [](double a, double b) { return a + b; });
        if (sum > 0) sc /= sum;
    }
    weight = (float)(sc * (double)r.scale);
}

template <int L, int PER, bool WIDE>
__global__ __launch_bounds__(256) void route_experts_kernel(const float *__restrict__ logits, int32_t *__restrict__ idx, float *__restrict__ w, int T, int E,
                                                            Routing r) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int ls = threadIdx.x % L;
    const int64_t t = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L, from = t < T ? t : T - 1;
    int chosen;
    float weight;
    route_token_lanes<L, PER, WIDE>(logits + from * E, E, r, lds, chosen, weight);
    if (t < T && ls < r.top_k) {
        idx[t * r.top_k + ls] = chosen;
        w[t * r.top_k + ls] = weight;
    }
}

// ---- sorting: each workgroup a chunk of pairs.  e: the thread's expert, or -1.  Returns how many pairs of the chunk in front of it have the same expert;
// s_cnt [16][E]: left as the counts of each wave's predecessors, s_total [E]: the chunk's pairs of each expert
__device__ __forceinline__ int chunk_rank(int e, int E, uint16_t *s_cnt, int32_t *s_total) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    for (int i = tid; i < waves * E; i += blockDim.x) s_cnt[i] = 0;
    __syncthreads();
    unsigned long long same = __ballot(e >= 0);
    for (int b = 0; 1 << b < E; ++b) {
        const unsigned long long m = __ballot(e >> b & 1);
        same &= e >> b & 1 ? m : ~m;
    }
    int rank = __popcll(same & ((1ull << lane) - 1));
    if (e >= 0 && rank == 0) s_cnt[wave * E + e] = (uint16_t)__popcll(same);
    __syncthreads();
    if (tid < E) {
        int n = 0;
        for (int i = 0; i < waves; ++i) {
            const int c = s_cnt[i * E + tid];
            s_cnt[i * E + tid] = (uint16_t)n;
            n += c;
        }
        s_total[tid] = n;
    }
    __syncthreads();
    return e >= 0 ? rank + s_cnt[wave * E + e] : 0;
}
// s_first[e] = sum of s_total in front of e, s_first[E] = all; by the first wave
__device__ __forceinline__ void experts_first(int E, const int32_t *s_total, int32_t *s_first) {
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int before = 0;
        for (int c = 0; c < E; c += 64) {
            const int v = c + lane < E ? s_total[c + lane] : 0;
            int upto = v;
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const int o = __shfl_up(upto, d);
                upto += lane >= d ? o : 0;
            }
            if (c + lane < E) s_first[c + lane] = before + upto - v;
            before += __shfl(upto, 63);
        }
        if (lane == 0) s_first[E] = before;
    }
    __syncthreads();
}

// Rows of the pairs.  COUNTED: the ranks inside a chunk and the chunks' counts are there (sort_count_kernel); else a workgroup counts all pairs itself, which is
// quicker than another launch up to some ten thousand of them.
__global__ __launch_bounds__(kSortChunk) void sort_count_kernel(const int32_t *__restrict__ idx, RouteSort s, int P, int E) {
    __shared__ uint16_t s_cnt[16 * kRouteExperts];
    __shared__ int32_t s_total[kRouteExperts];
    const int tid = threadIdx.x;
    const int64_t p = (int64_t)blockIdx.x * kSortChunk + tid;
    const int rank = chunk_rank(p < P ? idx[p] : -1, E, s_cnt, s_total);
    if (tid < E) s.hist[(int64_t)blockIdx.x * E + tid] = s_total[tid];
    if (p < P) s.pos[p] = rank;
}
template <bool COUNTED>
__global__ __launch_bounds__(kSortChunk) void sort_place_kernel(const int32_t *__restrict__ idx, RouteSort s, int P, int E, int top_k) {
    __shared__ uint16_t s_cnt[COUNTED ? 1 : 16 * kRouteExperts];
    __shared__ int32_t s_total[kRouteExperts], s_before[kRouteExperts], s_all[kRouteExperts], s_first[kRouteExperts + 1];
    const int tid = threadIdx.x;
    const int64_t chunk = (int64_t)blockIdx.x * kSortChunk, p = chunk + tid;
    const int e = p < P ? idx[p] : -1;
    int row = 0;
    if (COUNTED) {
        if (p < P) row = s.pos[p];
        if (tid < E) {
            int before = 0, all = 0;
            for (int c = 0; c < (int)gridDim.x; ++c) {
                const int n = s.hist[(int64_t)c * E + tid];
                before += c < (int)blockIdx.x ? n : 0;
                all += n;
            }
            s_before[tid] = before;
            s_all[tid] = all;
        }
        __syncthreads();
    } else {
        if (tid < E) s_before[tid] = s_all[tid] = 0;
        __syncthreads();
        for (int64_t i = tid; i < P; i += kSortChunk)
            if (i < chunk || i >= chunk + kSortChunk) atomicAdd((i < chunk ? s_before : s_all) + idx[i], 1);
        row = chunk_rank(e, E, s_cnt, s_total);  // (its barriers are the counts' too)
        if (tid < E) s_all[tid] += s_before[tid] + s_total[tid];
        __syncthreads();
    }
    experts_first(E, s_all, s_first);
    if (blockIdx.x == 0)
        for (int i = tid; i <= E; i += kSortChunk) s.offsets[i] = s_first[i];
    if (p < P) {
        row += s_before[e] + s_first[e];
        s.pos[p] = row;
        s.tok[row] = (int32_t)(p / top_k);
    }
}

// Few tokens: one workgroup routes them and sorts their pairs.
template <int L, int PER, bool WIDE>
__global__ __launch_bounds__(1024) void route_few_kernel(const float *__restrict__ logits, int32_t *__restrict__ idx, float *__restrict__ w, int T, int E, Routing r,
                                                         RouteSort s) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ uint16_t s_cnt[16 * kRouteExperts];
    __shared__ int32_t s_total[kRouteExperts], s_first[kRouteExperts + 1];
    __shared__ int16_t s_e[1024];
    const int tid = threadIdx.x, ls = tid % L, t = tid / L;
    s_e[tid] = -1;
    __syncthreads();
    int chosen;
    float weight;
    route_token_lanes<L, PER, WIDE>(logits + (int64_t)(t < T ? t : T - 1) * E, E, r, lds, chosen, weight);
    if (t < T && ls < r.top_k) {
        idx[t * r.top_k + ls] = chosen;
        w[t * r.top_k + ls] = weight;
        s_e[t * r.top_k + ls] = (int16_t)chosen;
    }
    __syncthreads();
    const int e = s_e[tid];
    int row = chunk_rank(e, E, s_cnt, s_total);
    experts_first(E, s_total, s_first);
    for (int i = tid; i <= E; i += blockDim.x) s.offsets[i] = s_first[i];
    if (e >= 0) {
        row += s_first[e];
        s.pos[tid] = row;
        s.tok[row] = tid / r.top_k;
    }
}

template <typename F>
static int with_shape(int E, bool wide, F f) {
    auto go = [&](auto l, auto per) {
        return wide ? f(l, per, std::true_type{}) : f(l, per, std::false_type{});
    };
#define CHADQ_INT(N) std::integral_constant<int, N>{}
    if (E <= 8) return go(CHADQ_INT(8), CHADQ_INT(1));
    if (E <= 16) return go(CHADQ_INT(16), CHADQ_INT(1));
    if (E <= 32) return go(CHADQ_INT(32), CHADQ_INT(1));
    if (E <= 64) return go(CHADQ_INT(64), CHADQ_INT(1));
    if (E <= 128) return go(CHADQ_INT(64), CHADQ_INT(2));
    if (E <= 256) return go(CHADQ_INT(64), CHADQ_INT(4));
    return go(CHADQ_INT(64), CHADQ_INT(8));
#undef CHADQ_INT
}

int route_experts_launch(const float *logits, int32_t *idx, float *w, int T, int E, const Routing &r, hipStream_t st) {
    return with_shape(E, r.bias || r.group_sum == 2, [&](auto l, auto per, auto wide) {
        constexpr int L = decltype(l)::value, PER = decltype(per)::value;
        constexpr bool WIDE = decltype(wide)::value;
        constexpr int tokens = 256 / L, most = tokens << 22;  // a launch has fewer than 2^32 threads
        const int lds = r.groups > 1 ? 256 * PER * (WIDE ? 8 : 4) : 0;
        for (int64_t t = 0; t < T; t += most) {
            const int n = (int)(T - t < most ? T - t : most);
            hipLaunchKernelGGL((route_experts_kernel<L, PER, WIDE>), dim3((n + tokens - 1) / tokens), dim3(256), lds, st, logits + t * E, idx + t * r.top_k, w + t * r.top_k, n, E, r);
            const int rc = hip_check(hipGetLastError(), "moe route launch");
            if (rc) return rc;
        }
        return 0;
    });
}

int route_sort_launch(const float *logits, int32_t *idx, float *w, int T, int E, const Routing &r, const RouteSort &s, hipStream_t st) {
    const int P = T * r.top_k, lanes = E <= 8 ? 8 : E <= 16 ? 16 : E <= 32 ? 32 : 64, most = E > 256 ? 512 : 1024;  // (threads: the groups' LDS)
    if ((int64_t)T * lanes <= most)
        return with_shape(E, r.bias || r.group_sum == 2, [&](auto l, auto per, auto wide) {
            constexpr int L = decltype(l)::value, PER = decltype(per)::value;
            constexpr bool WIDE = decltype(wide)::value;
            const int threads = T * L <= 256 && E <= 256 ? 256 : most, lds = r.groups > 1 ? threads * PER * (WIDE ? 8 : 4) : 0;
            hipLaunchKernelGGL((route_few_kernel<L, PER, WIDE>), dim3(1), dim3(threads), lds, st, logits, idx, w, T, E, r, s);
            return hip_check(hipGetLastError(), "moe route launch");
        });
    int rc = route_experts_launch(logits, idx, w, T, E, r, st);
    if (rc) return rc;
    const int chunks = sort_chunks(P);
    if (chunks <= kSortAlone) {
        hipLaunchKernelGGL(sort_place_kernel<false>, dim3(chunks), dim3(kSortChunk), 0, st, idx, s, P, E, r.top_k);
    } else {
        hipLaunchKernelGGL(sort_count_kernel, dim3(chunks), dim3(kSortChunk), 0, st, idx, s, P, E);
        hipLaunchKernelGGL(sort_place_kernel<true>, dim3(chunks), dim3(kSortChunk), 0, st, idx, s, P, E, r.top_k);
    }
    return hip_check(hipGetLastError(), "moe sort launch");
}

}  // namespace chadq
