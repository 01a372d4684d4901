// A token's rows from the experts, weighted and added to the residual stream, y[t] = r[t] + sum_j w[t, j] x[places[t, j]], and the gradients of rows and weights.
// Bound by the bytes of the rows, each read once.  Sums are kept in 32 bits, in the order of j, and rounded once.  Places outside of x count as none.
#ifndef TIRAMISU_AMD_COMBINE_HIP_H
#define TIRAMISU_AMD_COMBINE_HIP_H
#include "operator_elements.hip.h"

namespace tcombine {

using namespace tops;

struct combine_arguments {
    const void *x, *residual;               // residual: may be null
    const int *places;                      // [tokens][k]
    const float *weights;                   // [tokens][k], null: ones
    void *y;
    long tokens, rows, columns, ldx, ldr;   // rows: of x
    int k;
};

// 8 columns of a token to a thread; AHEAD rows are on their way at a time
template <int E>
__global__ __launch_bounds__(256) void combine_kernel(combine_arguments a) {
    constexpr int AHEAD = 8;
    const long across = (a.columns + 7) / 8, id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= across * a.tokens) return;
    const long t = id / across, n = 8 * (id - t * across);
    const long left = 2 * (a.columns - n);
    const int some = (int)min(8L, a.columns - n);
    typedef stored<E> T;
    u32x4 residual = {0, 0, 0, 0};
    if (a.residual) residual = load_to_end<2>((const char *)((const T *)a.residual + t * a.ldr + n), left, 2 * a.columns);
    float sum[8];
#pragma unroll
    for (int i = 0; i < 8; i++) sum[i] = 0.f;
    for (int j0 = 0; j0 < a.k; j0 += AHEAD) {
        u32x4 held[AHEAD];
        float w[AHEAD];
        bool there[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            const int place = j0 + j < a.k ? a.places[t * a.k + j0 + j] : -1;
            there[j] = place >= 0 && place < a.rows;
            w[j] = there[j] ? a.weights ? a.weights[t * a.k + j0 + j] : 1.f : 0.f;
            held[j] = u32x4{0, 0, 0, 0};
            if (there[j]) held[j] = load_to_end<2>((const char *)((const T *)a.x + place * a.ldx + n), left, 2 * a.columns);
        }
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            if (!there[j]) continue;
            float v[8];
            widen<E>(held[j], v);
#pragma unroll
            for (int i = 0; i < 8; i++) sum[i] = __builtin_fmaf(w[j], v[i], sum[i]);
        }
    }
    if (a.residual) {
        float r[8];
        widen<E>(residual, r);
#pragma unroll
        for (int i = 0; i < 8; i++) sum[i] += r[i];
    }
    store_some<E>((T *)a.y + t * a.columns + n, some, sum);
}

struct combine_backward_arguments {
    const void *dy, *x;
    const int *places, *owners;             // owners: the token of each row, negative: nobody's
    const float *weights;                   // null: ones, and no gradient of them
    void *dx;                               // dense, may be null
    float *dweights;                        // [tokens][k], may be null
    long tokens, rows, columns, ldy, ldx;
    int k;
    long token_blocks;
};

// THREADS to a token, of a workgroup of 256: its row of dy is read once for every four of its rows; behind the tokens' workgroups some that write nobody's rows.
template <int E, int THREADS>
__global__ __launch_bounds__(256) void combine_backward_kernel(combine_backward_arguments a) {
    constexpr int TEAMS = 256 / THREADS, AHEAD = 4, WAVES = THREADS / 64;
    typedef stored<E> T;
    __shared__ float sums[TEAMS][WAVES][AHEAD];
    const int team = threadIdx.x / THREADS, x = threadIdx.x % THREADS, lane = threadIdx.x & 63;
    if ((long)blockIdx.x >= a.token_blocks) {
        // 64 rows to a wavefront, whose lanes read their owners at once
        const long first = (((long)blockIdx.x - a.token_blocks) * 4 + threadIdx.x / 64) * 64, s = first + lane;
        const int owner = s < a.rows ? a.owners[s] : 0;
        for (unsigned long long none = __ballot(s < a.rows && (owner < 0 || owner >= a.tokens)); none; none &= none - 1) {
            const long row = first + __builtin_ctzll(none);
            const float zeros[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            for (long n = 8 * lane; n < a.columns; n += 512) store_some<E>((T *)a.dx + row * a.columns + n, (int)min(8L, a.columns - n), zeros);
        }
        return;
    }
    const long t = (long)blockIdx.x * TEAMS + team;
    const bool mine = t < a.tokens;
    for (int j0 = 0; j0 < a.k; j0 += AHEAD) {
        long place[AHEAD];
        float w[AHEAD], dot[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            const bool asked = mine && j0 + j < a.k;
            place[j] = asked ? a.places[t * a.k + j0 + j] : -1;
            if (place[j] >= a.rows) place[j] = -1;
            w[j] = !asked ? 0.f : a.weights ? a.weights[t * a.k + j0 + j] : 1.f;
            dot[j] = 0.f;
        }
        for (long n = 8 * x; mine && n < a.columns; n += 8 * THREADS) {
            const long left = 2 * (a.columns - n);
            const int some = (int)min(8L, a.columns - n);
            float d[8];
            const u32x4 held_d = load_to_end<2>((const char *)((const T *)a.dy + t * a.ldy + n), left, 2 * a.columns);
            u32x4 held[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; j++) {
                held[j] = u32x4{0, 0, 0, 0};
                if (a.dweights && place[j] >= 0) held[j] = load_to_end<2>((const char *)((const T *)a.x + place[j] * a.ldx + n), left, 2 * a.columns);
            }
            widen<E>(held_d, d);
#pragma unroll
            for (int j = 0; j < AHEAD; j++) {
                if (place[j] < 0) continue;
                float v[8], out[8];
                widen<E>(held[j], v);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    dot[j] = __builtin_fmaf(d[i], v[i], dot[j]);
                    out[i] = w[j] * d[i];
                }
                if (a.dx) store_some<E>((T *)a.dx + place[j] * a.columns + n, some, out);
            }
        }
        if (!a.dweights) continue;
#pragma unroll
        for (int j = 0; j < AHEAD; j++)
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) dot[j] += __shfl_xor(dot[j], o);
        if constexpr (WAVES > 1) {
            __syncthreads();
            if (lane == 0)
#pragma unroll
                for (int j = 0; j < AHEAD; j++) sums[team][x >> 6][j] = dot[j];
            __syncthreads();
#pragma unroll
            for (int j = 0; j < AHEAD; j++) {
                dot[j] = 0.f;
#pragma unroll
                for (int v = 0; v < WAVES; v++) dot[j] += sums[team][v][j];
            }
        }
#pragma unroll
        for (int j = 0; j < AHEAD; j++)
            if (mine && x == 0 && j0 + j < a.k) a.dweights[t * a.k + j0 + j] = place[j] >= 0 ? dot[j] : 0.f;
    }
}

}  // namespace tcombine
#endif
