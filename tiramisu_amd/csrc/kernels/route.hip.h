// A router's choice: the k best of a token's logits, their weights, and the tokens' places grouped by expert; and the gradient of the logits.
//
// LANES lanes of a wavefront hold the logits of a token, VALUES neighbouring ones each, as whole numbers that order them (zeros of either sign alike, NaN above
// everything).  A choice is the largest number over the lanes and then the lowest index that holds it.  Chosen
// ones become the least number; minus infinity is never chosen.  Sixteen lanes are one row of the cross-lane network, so that up to 256 experts take four tokens a wavefront
// without a word through LDS (200 experts, 16384 tokens: 29.8 us with a wavefront to a token, so 20).
//
// Places are counted, without atomics whose order could be seen: assignments, in order of token and rank, are the experts' in the order that they come.  Blocks of
// tokens count theirs while they choose; the second kernel adds the blocks before its own and ranks its own by ballots (a wavefront's lanes of one expert) and by
// sums over its wavefronts.  One workgroup does both for few tokens.
#ifndef TIRAMISU_AMD_ROUTE_HIP_H
#define TIRAMISU_AMD_ROUTE_HIP_H
#include <type_traits>

#include "operator_elements.hip.h"

namespace troute {

using namespace tops;

constexpr int MOST_EXPERTS = 1024, MOST_CHOSEN = 16;

struct route_arguments {
    const void *logits;
    long ld, tokens;
    int experts, k;
    int normalise;
    int *chosen;                            // [tokens][k]
    float *weights;                         // [tokens][k]
    int *offsets, *rows, *places;           // [experts + 1], [tokens k], [tokens][k]
    int *counts;                            // [blocks][experts], where there are several
    int block;                              // tokens of a block
};

// Orders like the number: NaN above all, zeros alike.  Never 0.
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.f);
    return v != v ? 0xffffffffu : u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float number_of(uint32_t o) {
    if (o == 0xffffffffu) return __builtin_nanf("");
    return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
constexpr uint32_t LEAST = 0x007fffffu;     // of minus infinity

// f over the LANES consecutive lanes that a lane belongs to, in each of them: within a row of 16 by turns of the cross-lane network, across rows by scalars
template <int LANES, class F, class T>
__device__ __forceinline__ T over_lanes(T v, F f) {
    static_assert(sizeof(T) == 4 && (LANES == 16 || LANES == 64), "rows of 16 lanes");
    auto turned = [](T x, auto by) {
        return __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x120 + decltype(by)::value, 0xf, 0xf, false));        // row_ror
    };
    v = f(v, turned(v, std::integral_constant<int, 8>()));
    v = f(v, turned(v, std::integral_constant<int, 4>()));
    v = f(v, turned(v, std::integral_constant<int, 2>()));
    v = f(v, turned(v, std::integral_constant<int, 1>()));
    if constexpr (LANES == 64) {
        auto of_row = [&](int lane) { return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); };
        return f(f(of_row(0), of_row(16)), f(of_row(32), of_row(48)));
    }
    return v;
}

// A lane's VALUES logits of a token; minus infinity behind the last
template <int E, int LANES, int VALUES>
__device__ __forceinline__ void load_logits(const void *logits, long ld, long token, int experts, int at, float (&v)[VALUES]) {
    const stored<E> *const row = (const stored<E> *)logits + token * ld + at * VALUES;
    const int some = experts - at * VALUES;
    if constexpr (VALUES * sizeof(stored<E>) % 16 == 0) {
        if (some >= VALUES) return load_elements<E>(row, v);
    }
#pragma unroll
    for (int i = 0; i < VALUES; i++) v[i] = i < some ? load_one<E>(row + i) : -__builtin_inff();
}

// Chooses for `token`; lane j of the LANES writes the j-th.  All lanes of the wavefront call it; `there`: whether the token exists.
template <int E, int LANES, int VALUES>
__device__ __forceinline__ void choose(const route_arguments &a, long token, bool there, int lane) {
    const int at = lane % LANES;
    float v[VALUES];
    uint32_t order[VALUES];
    load_logits<E, LANES, VALUES>(a.logits, a.ld, there ? token : 0, a.experts, at, v);
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < VALUES; i++) {
        order[i] = order_of(v[i]);
        best = max(best, order[i]);
    }
    int mine = -1;                                          // of rank `at`
    float z = 0.f, most = 0.f;
    for (int j = 0; j < a.k; j++) {
        const uint32_t top = over_lanes<LANES>(best, [](uint32_t x, uint32_t y) { return max(x, y); });
        int index = 0;
#pragma unroll
        for (int i = VALUES - 1; i >= 0; i--) index = order[i] == top ? i : index;
        index = over_lanes<LANES>(best == top ? at * VALUES + index : MOST_EXPERTS, [](int x, int y) { return min(x, y); });
        const int expert = top > LEAST ? index : -1;
        const float value = number_of(top);
        if (j == 0) most = expert >= 0 ? value : 0.f;
        if (at == j) { mine = expert; z = value; }
        best = 0;
#pragma unroll
        for (int i = 0; i < VALUES; i++) {
            if (at * VALUES + i == expert) order[i] = 0;
            best = max(best, order[i]);
        }
    }
    // exp(z - most): 0 for what was not chosen
    auto exponential = [&](float x) { return expf(x - most); };
    const float e = mine >= 0 ? exponential(z) : 0.f;
    float sum = e;
    if (!a.normalise) {
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < VALUES; i++) sum += v[i] == -__builtin_inff() ? 0.f : exponential(v[i]);
    }
    sum = over_lanes<LANES>(sum, [](float x, float y) { return x + y; });
    if (there && at < a.k) {
        a.chosen[token * a.k + at] = mine;
        a.weights[token * a.k + at] = mine >= 0 ? e / sum : 0.f;
    }
}

// Ranks the assignments first .. end - 1 of a.chosen, in their order, behind `next` of each expert (in LDS; moved on), and writes their places.
// hist: [wavefronts][experts] in LDS.  All threads of the workgroup call it.
template <int THREADS, typename INTS>
__device__ __forceinline__ void place(const route_arguments &a, long first, long end, INTS next, INTS hist) {
    constexpr int WAVES = THREADS / 64;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    for (long from = first; from < end; from += THREADS) {
        for (int i = t; i < WAVES * a.experts; i += THREADS) hist[i] = 0;
        __syncthreads();
        const long i = from + t;
        const int e = i < end ? a.chosen[i] : -1;
        // lanes of the same expert, by the bits of its number (those without one apart: the bit above)
        unsigned long long same = __ballot(e >= 0);
        same = e >= 0 ? same : ~same;
        for (int bit = 1; bit < a.experts; bit *= 2) {
            const unsigned long long with = __ballot((e & bit) != 0);
            same &= e & bit ? with : ~with;
        }
        const int before = __popcll(same & ((1ull << lane) - 1));
        if (e >= 0 && before == 0) hist[wave * a.experts + e] = __popcll(same);
        __syncthreads();
        if (e >= 0) {
            int at = next[e] + before;
            for (int w = 0; w < wave; w++) at += hist[w * a.experts + e];
            a.places[i] = at;
            a.rows[at] = (int)(i / a.k);
        } else if (i < end) a.places[i] = -1;
        if (from + THREADS >= end) break;
        __syncthreads();
        for (int x = t; x < a.experts; x += THREADS)
            for (int w = 0; w < WAVES; w++) next[x] += hist[w * a.experts + x];
        __syncthreads();
    }
}

// next[e] = sum of counts of the experts before, for up to 1024 experts; returns the sum of all.  `sums`: an int for each wavefront.
template <int THREADS, typename INTS>
__device__ __forceinline__ int sum_before(int experts, INTS count, INTS sums) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    constexpr int WAVES = THREADS / 64, EACH = MOST_EXPERTS / THREADS;
    int v[EACH], own = 0;
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const int e = t * EACH + i;
        v[i] = own;
        own += e < experts ? count[e] : 0;
    }
    int upto = own;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const int from = __shfl_up(upto, o);
        if (lane >= o) upto += from;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        const int s = sums[w];
        if (w < wave) base += s;
        all += s;
    }
#pragma unroll
    for (int i = 0; i < EACH; i++)
        if (t * EACH + i < experts) count[t * EACH + i] = base + upto - own + v[i];
    __syncthreads();
    return all;
}

constexpr int ROUTE_THREADS = 1024, ROUTE_FEW_THREADS = 512;
typedef __attribute__((address_space(3))) int lds_int;
inline int route_lds_bytes(int experts, int threads) { return ((threads / 64 + 2) * experts + 64) * 4; }

template <int E, int LANES, int VALUES, int THREADS>
__device__ __forceinline__ void choose_block(const route_arguments &a, long first, long end) {
    constexpr int TOKENS = THREADS / LANES;
    for (long from = first; from < end; from += TOKENS) {
        const long token = from + threadIdx.x / LANES;
        choose<E, LANES, VALUES>(a, token, token < end, threadIdx.x & 63);
    }
}

// Everything, for few tokens: one workgroup
template <int E, int LANES, int VALUES>
__global__ __launch_bounds__(ROUTE_FEW_THREADS) void route_few_kernel(route_arguments a) {
    extern __shared__ __attribute__((aligned(16))) char shared_bytes[];
    lds_int *const next = (lds_int *)shared_bytes, *const hist = next + a.experts, *const sums = hist + ROUTE_FEW_THREADS / 64 * a.experts;
    const int t = threadIdx.x;
    for (int e = t; e < a.experts; e += ROUTE_FEW_THREADS) next[e] = 0;
    choose_block<E, LANES, VALUES, ROUTE_FEW_THREADS>(a, 0, a.tokens);
    __syncthreads();
    const long all = a.tokens * a.k;
    for (long i = t; i < all; i += ROUTE_FEW_THREADS) {
        const int e = a.chosen[i];
        if (e >= 0) __hip_atomic_fetch_add(next + e, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
    __syncthreads();
    const int total = sum_before<ROUTE_FEW_THREADS>(a.experts, next, sums);
    for (int e = t; e < a.experts; e += ROUTE_FEW_THREADS) a.offsets[e] = next[e];
    if (t == 0) a.offsets[a.experts] = total;
    __syncthreads();
    place<ROUTE_FEW_THREADS>(a, 0, all, next, hist);
    for (long i = total + t; i < all; i += ROUTE_FEW_THREADS) a.rows[i] = -1;
}

// A block of tokens: their choices, and how many of each expert
template <int E, int LANES, int VALUES>
__global__ __launch_bounds__(ROUTE_THREADS) void route_choose_kernel(route_arguments a) {
    extern __shared__ __attribute__((aligned(16))) char shared_bytes[];
    lds_int *const count = (lds_int *)shared_bytes;
    const int t = threadIdx.x;
    const long first = (long)blockIdx.x * a.block, end = min(first + a.block, a.tokens);
    for (int e = t; e < a.experts; e += ROUTE_THREADS) count[e] = 0;
    choose_block<E, LANES, VALUES, ROUTE_THREADS>(a, first, end);
    __syncthreads();
    for (long i = first * a.k + t; i < end * a.k; i += ROUTE_THREADS) {
        const int e = a.chosen[i];
        if (e >= 0) __hip_atomic_fetch_add(count + e, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
    __syncthreads();
    for (int e = t; e < a.experts; e += ROUTE_THREADS) a.counts[(long)blockIdx.x * a.experts + e] = count[e];
}

// ... their places
__global__ __launch_bounds__(ROUTE_THREADS) void route_place_kernel(route_arguments a) {
    extern __shared__ __attribute__((aligned(16))) char shared_bytes[];
    lds_int *const next = (lds_int *)shared_bytes, *const hist = next + a.experts, *const sums = hist + ROUTE_THREADS / 64 * a.experts, *const before = sums + 64;
    const int t = threadIdx.x, blocks = gridDim.x;
    const long first = (long)blockIdx.x * a.block, end = min(first + a.block, a.tokens);
    for (int e = t; e < 2 * a.experts; e += ROUTE_THREADS) (e < a.experts ? next[e] : before[e - a.experts]) = 0;
    __syncthreads();
    // sums over the blocks, and over those before this one: threads that share an expert take blocks in turn
    const int sharers = max(1, ROUTE_THREADS / a.experts);
    for (int w = t; w < sharers * a.experts; w += ROUTE_THREADS) {
        const int e = w % a.experts;
        int all = 0, early = 0;
#pragma unroll 16
        for (int b = w / a.experts; b < blocks; b += sharers) {
            const int c = a.counts[(long)b * a.experts + e];
            all += c;
            early += b < (int)blockIdx.x ? c : 0;
        }
        __hip_atomic_fetch_add(next + e, all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        __hip_atomic_fetch_add(before + e, early, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
    __syncthreads();
    const int total = sum_before<ROUTE_THREADS>(a.experts, next, sums);
    if (blockIdx.x == 0) {
        for (int e = t; e < a.experts; e += ROUTE_THREADS) a.offsets[e] = next[e];
        if (t == 0) a.offsets[a.experts] = total;
    }
    __syncthreads();
    for (int e = t; e < a.experts; e += ROUTE_THREADS) next[e] += before[e];
    __syncthreads();
    place<ROUTE_THREADS>(a, first * a.k, end * a.k, next, hist);
    for (long i = max((long)total, first * a.k) + t; i < end * a.k; i += ROUTE_THREADS) a.rows[i] = -1;
}

// ---- the gradient of the logits.  w_j = e_j / sum, e = exp(z - most); normalised (the sum over the chosen): dz_j = w_j (g_j - sum_i g_i w_i); over all: also - p_e sum_i
// g_i w_i for every expert e.  An expert that is chosen twice has both terms.
struct route_backward_arguments {
    const float *dweights;
    const void *logits;
    const int *chosen;
    void *dlogits;                          // dense
    long ld, tokens;
    int experts, k, normalise;
};
template <int E, int LANES, int VALUES>
__global__ __launch_bounds__(256) void route_backward_kernel(route_backward_arguments a) {
    const int lane = threadIdx.x & 63, at = lane % LANES, base = lane - at;
    const long token = (long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const bool there = token < a.tokens;
    const long row = there ? token : 0;
    float v[VALUES];
    load_logits<E, LANES, VALUES>(a.logits, a.ld, row, a.experts, at, v);
    int expert = -1;
    float g = 0.f, z = -__builtin_inff();
    if (at < a.k) {
        expert = a.chosen[row * a.k + at];
        if (expert < 0 || expert >= a.experts) expert = -1;
        if (expert >= 0) {
            g = a.dweights[row * a.k + at];
            z = load_one<E>((const stored<E> *)a.logits + row * a.ld + expert);
        }
    }
    // the largest of those that the sum is over; a NaN among them makes the whole row one, as in the forward pass
    auto larger = [](float x, float y) { return x != x || y != y ? x + y : max(x, y); };
    float most = a.normalise ? z : v[0];
#pragma unroll
    for (int i = 1; i < VALUES; i++) most = a.normalise ? most : larger(most, v[i]);
    most = over_lanes<LANES>(most, larger);
    const bool any = over_lanes<LANES>((int)(expert >= 0), [](int x, int y) { return x | y; }) != 0;
    if (!any) most = 0.f;
    const float e = expert >= 0 ? expf(z - most) : 0.f;
    float all[VALUES], sum = a.normalise ? e : 0.f;
#pragma unroll
    for (int i = 0; i < VALUES; i++) {
        all[i] = a.normalise || v[i] == -__builtin_inff() ? 0.f : expf(v[i] - most);
        sum += all[i];
    }
    auto add = [](float x, float y) { return x + y; };
    sum = over_lanes<LANES>(sum, add);
    const float share = any ? 1.f / sum : 0.f, w = expert >= 0 ? e * share : 0.f;
    const float dot = over_lanes<LANES>(expert >= 0 ? w * g : 0.f, add);
    const float term = expert < 0 ? 0.f : a.normalise ? w * (g - dot) : w * g;
    float out[VALUES];
#pragma unroll
    for (int i = 0; i < VALUES; i++) out[i] = a.normalise || !any || v[i] == -__builtin_inff() ? 0.f : -all[i] * share * dot;
    for (int j = 0; j < a.k; j++) {
        const int x = __shfl(expert, base + j);
        const float d = __shfl(term, base + j);
#pragma unroll
        for (int i = 0; i < VALUES; i++)
            if (at * VALUES + i == x) out[i] += d;
    }
    if (!there) return;
    stored<E> *const to = (stored<E> *)a.dlogits + token * a.experts;
#pragma unroll
    for (int i = 0; i < VALUES; i++)
        if (at * VALUES + i < a.experts) store_one<E>(to + at * VALUES + i, out[i]);
}

}  // namespace troute
#endif
