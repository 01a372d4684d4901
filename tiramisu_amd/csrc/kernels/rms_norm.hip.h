// Root-mean-square norm of rows, with the addition of a residual ahead of it and rows of 8-bit numbers with a scale behind it:
//     s = x + r,   rstd = 1 / sqrt(mean(s^2) + eps),   y = s rstd w,   or   q = e4m3(y / scale), scale = max|y| / 448
// and backward, from the gradient dy of y and ds that arrives along the residual stream:
//     dx = rstd (g - s rstd^2 mean(g s)) + ds with g = dy w,      dw = sum over rows of dy s rstd.
// Each input is read once and each output written once: a row stays in the registers of its team (64, 256 or 1024 threads, PER
// pieces of 16 bytes of the widest input each), which reduces it by lane exchanges and, where it is more than a wavefront, through LDS.  The norm
// is of the unrounded sum.  Rows too long for that are read a second time.
// Bound by the bytes: 16384 x 4096 bf16 with a residual 96 us, 5.6 TB/s (the fastest copy of 4 GiB: 5.5), to 8 bits 91, 5.1 TB/s, without a norm 51, 4.0;
// 8192 x 2048 backward 29.5 us, 4.5 TB/s, of which the sums' launch is 4.7.  Few rows are bound by the launch: one of 4096 to 8 bits 4.8 us, of which an empty kernel is 2.8.  Tried and not faster: weights
// loaded ahead of the reduction (100 us), a wavefront to a row forward.
// Sums of the backward pass over rows are kept per team in registers, written once a workgroup, and added by a second launch in a fixed
// order: results do not depend on the order of workgroups.
#ifndef TIRAMISU_AMD_RMS_NORM_HIP_H
#define TIRAMISU_AMD_RMS_NORM_HIP_H
#include "operator_elements.hip.h"

namespace tops {

struct norm_arguments {
    const void *x, *residual, *weight;      // residual: may be null; weight: null for quantize_rows
    void *y, *sum;                          // sum: may be null
    float *scale, *rstd;                    // may be null
    long rows, columns, ldx, ldr;
    float eps;
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// the larger of two, and NaN where one is
__device__ __forceinline__ float max_or_nan(float a, float b) { return a > b || a != a ? a : b; }
__device__ __forceinline__ float wave_max_or_nan(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max_or_nan(v, __shfl_xor(v, o));
    return v;
}

// Reductions over a team of TEAM threads.  `slot`: TEAM / 64 floats of LDS that no other reduction in flight uses; a team larger than a
// wavefront is the whole workgroup, and its slots alternate, so that one barrier a reduction is enough.
template <int TEAM, bool MAX>
__device__ __forceinline__ float team_reduce(float v, float *slot) {
    v = MAX ? wave_max_or_nan(v) : wave_sum(v);
    if constexpr (TEAM > 64) {
        constexpr int WAVES = TEAM / 64;
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        if (lane == 0) slot[wave] = v;
        __syncthreads();
        v = slot[lane & (WAVES - 1)];
#pragma unroll
        for (int o = WAVES / 2; o > 0; o >>= 1) {
            const float other = __shfl_xor(v, o);
            v = MAX ? max_or_nan(v, other) : v + other;
        }
    }
    return v;
}

// Y: element type of y (E, or F8).  HELD: the row fits TEAM x PER pieces; else it is read again.
template <int E, int Y, int TEAM, int PER, bool HELD>
__global__ __launch_bounds__(TEAM < 256 ? 256 : TEAM) void rms_norm_kernel(norm_arguments a) {
    constexpr int N = E == F32 ? 4 : 8;                      // elements of a piece
    constexpr int TEAMS = TEAM < 256 ? 256 / TEAM : 1;
    __shared__ float slots[2][TEAM > 64 ? TEAM / 64 : 1];
    const int t = threadIdx.x % TEAM;
    const long row = (long)blockIdx.x * TEAMS + threadIdx.x / TEAM;
    if (TEAMS > 1 && row >= a.rows) return;                  // a whole wavefront, and no barrier follows in teams of one
    typedef stored<E> T;
    const T *x = (const T *)a.x + row * a.ldx, *r = a.residual ? (const T *)a.residual + row * a.ldr : nullptr, *w = (const T *)a.weight;
    T *sum = a.sum ? (T *)a.sum + row * a.columns : nullptr;
    stored<Y> *y = (stored<Y> *)a.y + row * a.columns;
    const int pieces = HELD ? PER : (int)((a.columns + TEAM * N - 1) / (TEAM * N));

    float held[HELD ? PER : 1][N];
    float squares = 0.f;
    auto read = [&](int p, float (&v)[N]) {
        const long c = ((long)p * TEAM + t) * N;
        const int n = (int)min((long)N, a.columns - c);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = 0.f;
        if (n <= 0) return;
        load_some<E>(x + c, n, v);
        if (r) {
            float other[N];
            load_some<E>(r + c, n, other);
#pragma unroll
            for (int i = 0; i < N; i++) v[i] += other[i];
        }
    };
    auto finish = [&](int p, float (&v)[N], float factor) {  // v: s; becomes y
        const long c = ((long)p * TEAM + t) * N;
        const int n = (int)min((long)N, a.columns - c);
        if (!w || n <= 0) return;                            // (what lies behind the row is zero)
        float g[N];
        load_some<E>(w + c, n, g);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = v[i] * factor * g[i];
    };
    auto write_sum = [&](int p, float (&v)[N]) {
        const long c = ((long)p * TEAM + t) * N;
        const int n = (int)min((long)N, a.columns - c);
        if (n > 0) store_some<E>(sum + c, n, v);
    };

    if constexpr (HELD) {
#pragma unroll
        for (int p = 0; p < PER; p++) read(p, held[p]);
#pragma unroll
        for (int p = 0; p < PER; p++) {
#pragma unroll
            for (int i = 0; i < N; i++) squares += held[p][i] * held[p][i];
            if (sum) write_sum(p, held[p]);
        }
    } else {
        for (int p = 0; p < pieces; p++) {
            float v[N];
            read(p, v);
#pragma unroll
            for (int i = 0; i < N; i++) squares += v[i] * v[i];
        }
    }
    float rstd = 1.f;
    if (w) {
        squares = team_reduce<TEAM, false>(squares, slots[0]);
        rstd = 1.f / sqrtf(squares / (float)a.columns + a.eps);
        if (a.rstd && t == 0) a.rstd[row] = rstd;
    }
    float most = 0.f;
    if constexpr (Y == F8) {
        if constexpr (HELD) {
#pragma unroll
            for (int p = 0; p < PER; p++) {
                finish(p, held[p], rstd);
#pragma unroll
                for (int i = 0; i < N; i++) most = max_or_nan(fabsf(held[p][i]), most);
            }
        } else {
            for (int p = 0; p < pieces; p++) {
                float v[N];
                read(p, v);
                finish(p, v, rstd);
#pragma unroll
                for (int i = 0; i < N; i++) most = max_or_nan(fabsf(v[i]), most);
            }
        }
        most = team_reduce<TEAM, true>(most, slots[1]);
        most = most / E4M3_MOST;                             // the scale
        if (most == 0.f) most = 1.f;                         // of a row of zeros, or of numbers so small that their scale would be zero
        if (t == 0) a.scale[row] = most;
    }
    auto write = [&](int p, float (&v)[N]) {
        const long c = ((long)p * TEAM + t) * N;
        const int n = (int)min((long)N, a.columns - c);
        if (n <= 0) return;
        if constexpr (Y == F8) {
            // (a scale below the normal numbers is rounded coarsely: what then lies beyond the format's largest number is set to it; one that would be zero is 1)
#pragma unroll
            for (int i = 0; i < N; i++) {
                v[i] /= most;
                v[i] = v[i] > E4M3_MOST ? E4M3_MOST : v[i] < -E4M3_MOST ? -E4M3_MOST : v[i];
            }
        }
        store_some<Y>(y + c, n, v);
    };
    if constexpr (HELD) {
#pragma unroll
        for (int p = 0; p < PER; p++) {
            if constexpr (Y != F8) finish(p, held[p], rstd);
            write(p, held[p]);
        }
    } else {
        for (int p = 0; p < pieces; p++) {
            float v[N];
            read(p, v);
            if (sum) write_sum(p, v);
            finish(p, v, rstd);
            write(p, v);
        }
    }
}

struct norm_backward_arguments {
    const void *dy, *sum, *weight, *dsum;   // dsum: may be null
    const float *rstd;
    void *dx;
    float *partial;                         // [workgroups][columns]
    long rows, columns, ldy, lds, ldd;
    int parts;                              // (rows that no team holds: of the walk down the columns)
    long first;                             // (... and the launch's first row)
};

// Teams walk over the rows, team g taking rows g, g + teams, ....  Teams of one wavefront need no barrier on the way, and the eight of a workgroup add their
// columns' sums in LDS before they are written (8192 x 2048 bf16: workgroups of one team of 256 threads, a barrier a row, 44.5 us).
template <int E, int TEAM, int PER>
constexpr int norm_backward_threads = TEAM == 64 ? 512 : TEAM;
template <int E, int TEAM, int PER>
__global__ __launch_bounds__((norm_backward_threads<E, TEAM, PER>)) void rms_norm_backward_kernel(norm_backward_arguments a) {
    constexpr int N = E == F32 ? 4 : 8;
    constexpr int TEAMS = norm_backward_threads<E, TEAM, PER> / TEAM;
    __shared__ float slots[2][TEAM > 64 ? TEAM / 64 : 1];
    typedef stored<E> T;
    const int t = threadIdx.x % TEAM;
    const long team = (long)blockIdx.x * TEAMS + threadIdx.x / TEAM, teams = (long)gridDim.x * TEAMS;
    float dw[PER][N];
#pragma unroll
    for (int p = 0; p < PER; p++)
#pragma unroll
        for (int i = 0; i < N; i++) dw[p][i] = 0.f;
    // (pieces stay as they are in memory, a quarter or half of what they are as fp32, so that more rows are on their way in a compute unit)
    auto read = [&](const T *from, int p) {
        const long c = ((long)p * TEAM + t) * N;
        return load_guarded<sizeof(T)>((const char *)(from + c), (a.columns - c) * (long)sizeof(T));
    };
    u32x4 weights[PER];
#pragma unroll
    for (int p = 0; p < PER; p++) weights[p] = read((const T *)a.weight, p);
    int turn = 0;
    for (long row = team; row < a.rows; row += teams, turn ^= 1) {
        const T *dy = (const T *)a.dy + row * a.ldy, *s = (const T *)a.sum + row * a.lds, *ds = a.dsum ? (const T *)a.dsum + row * a.ldd : nullptr;
        const float rstd = a.rstd[row];
        u32x4 held_s[PER], held_dy[PER], held_ds[PER];
#pragma unroll
        for (int p = 0; p < PER; p++) asm volatile("" : "+v"(weights[p]));     // (not kept as fp32 from row to row: 32 registers more)
#pragma unroll
        for (int p = 0; p < PER; p++) {
            held_s[p] = read(s, p);
            held_dy[p] = read(dy, p);
        }
#pragma unroll
        for (int p = 0; p < PER; p++) held_ds[p] = ds ? read(ds, p) : u32x4{0, 0, 0, 0};
        float dot = 0.f;
#pragma unroll
        for (int p = 0; p < PER; p++) {
            float x[N], g[N], f[N];
            widen<E>(held_s[p], x);
            widen<E>(held_dy[p], g);
            widen<E>(weights[p], f);
#pragma unroll
            for (int i = 0; i < N; i++) {
                x[i] *= rstd;
                dw[p][i] += g[i] * x[i];
                dot += g[i] * f[i] * x[i];
            }
        }
        dot = team_reduce<TEAM, false>(dot, slots[turn]) / (float)a.columns;
        T *dx = (T *)a.dx + row * a.columns;
#pragma unroll
        for (int p = 0; p < PER; p++) {
            const long c = ((long)p * TEAM + t) * N;
            const int n = (int)min((long)N, a.columns - c);
            if (n <= 0) continue;
            float x[N], g[N], f[N], d[N];
            widen<E>(held_s[p], x);
            widen<E>(held_dy[p], g);
            widen<E>(weights[p], f);
            widen<E>(held_ds[p], d);
#pragma unroll
            for (int i = 0; i < N; i++) d[i] += rstd * (g[i] * f[i] - x[i] * rstd * dot);
            store_some<E>(dx + c, n, d);
        }
    }
    if constexpr (TEAMS > 1) {
        // one wavefront after the other, in order
        __shared__ float sums[PER][N][64];
        const int wave = threadIdx.x / 64;
        for (int turn_of = 0; turn_of < TEAMS; turn_of++) {
            if (wave == turn_of) {
#pragma unroll
                for (int p = 0; p < PER; p++)
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        if (turn_of > 0) dw[p][i] += sums[p][i][t];
                        if (turn_of < TEAMS - 1) sums[p][i][t] = dw[p][i];
                    }
            }
            __syncthreads();
        }
        if (wave != TEAMS - 1) return;
    }
#pragma unroll
    for (int p = 0; p < PER; p++) {
        const long c = ((long)p * TEAM + t) * N;
        const int n = (int)min((long)N, a.columns - c);
        if (n > 0) store_some<F32>(a.partial + (long)blockIdx.x * a.columns + c, n, dw[p]);
    }
}

// Rows that no team holds: dx by a workgroup for each row, reading it twice, and the columns' sums by threads that walk down them.
template <int E>
__global__ __launch_bounds__(1024) void rms_norm_backward_long_rows_kernel(norm_backward_arguments a) {
    __shared__ float slots[16];
    typedef stored<E> T;
    const long row = a.first + blockIdx.x;
    const T *dy = (const T *)a.dy + row * a.ldy, *s = (const T *)a.sum + row * a.lds, *w = (const T *)a.weight;
    const T *ds = a.dsum ? (const T *)a.dsum + row * a.ldd : nullptr;
    const float rstd = a.rstd[row];
    float dot = 0.f;
    for (long c = threadIdx.x; c < a.columns; c += 1024) dot += (float)dy[c] * (float)w[c] * ((float)s[c] * rstd);
    dot = team_reduce<1024, false>(dot, slots) / (float)a.columns;
    for (long c = threadIdx.x; c < a.columns; c += 1024) {
        float v = rstd * ((float)dy[c] * (float)w[c] - (float)s[c] * rstd * dot);
        if (ds) v += (float)ds[c];
        ((T *)a.dx)[row * a.columns + c] = (T)v;
    }
}
template <int E>
__global__ __launch_bounds__(256) void rms_norm_backward_long_columns_kernel(norm_backward_arguments a) {
    typedef stored<E> T;
    const long c = (long)blockIdx.x * 256 + threadIdx.x;
    if (c >= a.columns) return;
    float sum = 0.f;
    for (long row = blockIdx.y; row < a.rows; row += a.parts)
        sum += (float)((const T *)a.dy)[row * a.ldy + c] * ((float)((const T *)a.sum)[row * a.lds + c] * a.rstd[row]);
    a.partial[(long)blockIdx.y * a.columns + c] = sum;
}

template <int E>
__global__ __launch_bounds__(1024) void sum_parts_kernel(column_sums a) {
    __shared__ float s[1024 + 32];
    sum_parts<E, 1024>(a, blockIdx.x, s);
}

}  // namespace tops
#endif
