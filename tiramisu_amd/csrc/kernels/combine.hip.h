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
    long choice_blocks;
};

// LANES to a choice of a token: its row, and the token's row of dy, which the choices of a token, next to each other, share in the caches; no sums leave the lanes.  (A
// workgroup to a token, that reads dy once for all its choices, is behind its sums through LDS and its registers: 2000 x 3 x 1430 f16 13.3 us, so 10.5.)  Behind the choices'
// workgroups some that write nobody's rows.
template <int E, int LANES>
__global__ __launch_bounds__(256) void combine_backward_kernel(combine_backward_arguments a) {
    constexpr int AHEAD = 4;                               // pieces of either row on their way at a time
    typedef stored<E> T;
    const int lane = threadIdx.x & 63, at = threadIdx.x % LANES;
    if ((long)blockIdx.x >= a.choice_blocks) {
        // 16 rows to a wavefront, whose lanes read their owners at once; LANES to a row
        const long first = (((long)blockIdx.x - a.choice_blocks) * 4 + threadIdx.x / 64) * 16, s = first + lane % 16;
        const int owner = s < a.rows ? a.owners[s] : -1;
        bool written = false;                              // (the four lanes of a row share its token's choices)
        if (owner >= 0 && owner < a.tokens)
            for (int j = lane / 16; j < a.k; j += 4) written = written || a.places[(long)owner * a.k + j] == s;
        written = __shfl_xor((int)written, 16) || written;
        written = __shfl_xor((int)written, 32) || written;
        const bool none = s < a.rows && !written;
        for (int i = lane / LANES; i < 16; i += 64 / LANES) {
            const float zeros[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (!__shfl((int)none, i)) continue;
            for (long n = 8 * at; n < a.columns; n += 8 * LANES) store_some<E>((T *)a.dx + (first + i) * a.columns + n, (int)min(8L, a.columns - n), zeros);
        }
        return;
    }
    const long choice = (long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const bool there = choice < a.tokens * a.k;
    const int place = there ? a.places[choice] : -1;
    const bool mine = place >= 0 && place < a.rows;
    const float w = mine && a.weights ? a.weights[choice] : 1.f;
    float dot = 0.f;
    if (mine) {
        const T *const dy = (const T *)a.dy + choice / a.k * a.ldy, *const x = (const T *)a.x + (long)place * a.ldx;
        T *const dx = (T *)a.dx + (long)place * a.columns;
        for (long n0 = 8 * at; n0 < a.columns; n0 += 8 * LANES * AHEAD) {
            u32x4 held_d[AHEAD], held_x[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const long n = n0 + 8 * LANES * i, left = 2 * (a.columns - n);
                held_d[i] = held_x[i] = u32x4{0, 0, 0, 0};
                if (left <= 0) continue;
                held_d[i] = load_to_end<2>((const char *)(dy + n), left, 2 * a.columns);
                if (a.dweights) held_x[i] = load_to_end<2>((const char *)(x + n), left, 2 * a.columns);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const long n = n0 + 8 * LANES * i;
                if (n >= a.columns) continue;
                float d[8], v[8];
                widen<E>(held_d[i], d);
                widen<E>(held_x[i], v);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    dot = __builtin_fmaf(d[e], v[e], dot);
                    d[e] *= w;
                }
                if (a.dx) store_some<E>(dx + n, (int)min(8L, a.columns - n), d);
            }
        }
    }
    if (!a.dweights) return;
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) dot += __shfl_xor(dot, o);
    if (there && at == 0) a.dweights[choice] = dot;
}

}  // namespace tcombine
#endif
