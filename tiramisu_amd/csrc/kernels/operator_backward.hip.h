// Elementwise parts of the operators' backward passes, and rows moved to where the tiles can load them.  Bound by the bytes they move; one thread
// takes 8 elements of a row at a time.
#ifndef TIRAMISU_AMD_OPERATOR_BACKWARD_HIP_H
#define TIRAMISU_AMD_OPERATOR_BACKWARD_HIP_H
#include "operator_elements.hip.h"

namespace tops {

struct activation_backward_arguments {
    const void *dy, *pre;                   // pre: null where there is no activation
    void *dz;                               // may be null
    float *partial;                         // [chunks][N], may be null: column sums of dz, ahead of its rounding
    long M, N, ldy, ldp, ldz, rows;         // rows: of a chunk
    int activation, across;                 // across: threads along a row, a power of two
};

// dz = dy activation'(pre), and its sums over the rows of a chunk (the bias's gradient; the chunks are added by sum_parts_kernel).
// dz is rounded to the operands' 16 bits, as it is multiplied by matrix instructions of that type.
// 4096 x 4096 bf16 with gelu: 21.4 us, 4.7 TB/s (one row at a time 24); 300 x 520 with one row to a thread 3.4 us less than with four.
template <int E>
__global__ __launch_bounds__(256) void activation_backward_kernel(activation_backward_arguments a) {
    __shared__ float s[256][9];
    const int x = threadIdx.x & (a.across - 1), y = threadIdx.x / a.across, down = 256 / a.across;
    const long n = ((long)blockIdx.x * a.across + x) * 8;
    const int some = (int)max(0L, min(8L, a.N - n));
    const long end = min(a.M, (long)(blockIdx.y + 1) * a.rows);
    typedef stored<E> T;
    float sum[8];
#pragma unroll
    for (int i = 0; i < 8; i++) sum[i] = 0.f;
    if (some > 0) {
        // (ROWS rows are on their way at a time)
        constexpr int ROWS = 4;
        for (long m = (long)blockIdx.y * a.rows + y; m < end; m += ROWS * down) {
            u32x4 held[ROWS], held_pre[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                const long row = m + r * down, left = row < end ? 2 * some : 0;
                held[r] = load_guarded<2>((const char *)((const T *)a.dy + row * a.ldy + n), left);
                if (a.pre) held_pre[r] = load_guarded<2>((const char *)((const T *)a.pre + row * a.ldp + n), left);
            }
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                const long row = m + r * down;
                if (row >= end) break;
                float v[8];
                widen<E>(held[r], v);
                if (a.pre) {
                    float z[8], slope[8], value[8];
                    widen<E>(held_pre[r], z);
                    activation_slopes(a.activation, z, slope, value);
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] *= slope[i];
                }
                if (a.dz) store_some<E>((T *)a.dz + row * a.ldz + n, some, v);
#pragma unroll
                for (int i = 0; i < 8; i++) sum[i] += v[i];
            }
        }
    }
    if (!a.partial) return;
#pragma unroll
    for (int i = 0; i < 8; i++) s[threadIdx.x][i] = sum[i];
    __syncthreads();
    if (y != 0 || some == 0) return;
    for (int r = 1; r < down; r++)
#pragma unroll
        for (int i = 0; i < 8; i++) sum[i] += s[r * a.across + x][i];
    store_some<F32>(a.partial + (long)blockIdx.y * a.N + n, some, sum);
}

struct gated_backward_arguments {
    const void *dh, *gate, *up;
    void *dgate, *dup;                      // rows of ldd
    long M, N, ldh, ldg, ldu, ldd;
    int activation;
};

// dgate = dh up activation'(gate), dup = dh activation(gate): 16 bits as they are multiplied.  4096 x 4096 bf16: 30 us, 5.6 TB/s.
template <int E>
__global__ __launch_bounds__(256) void gated_backward_kernel(gated_backward_arguments a) {
    const long across = (a.N + 7) / 8, id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= across * a.M) return;
    const long m = id / across, n = 8 * (id - m * across);
    const int some = (int)min(8L, a.N - n);
    typedef stored<E> T;
    float d[8], g[8], u[8];
    load_some<E>((const T *)a.dh + m * a.ldh + n, some, d);
    load_some<E>((const T *)a.gate + m * a.ldg + n, some, g);
    load_some<E>((const T *)a.up + m * a.ldu + n, some, u);
    float slope[8], value[8];
    activation_slopes(a.activation, g, slope, value);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        g[i] = d[i] * u[i] * slope[i];
        u[i] = d[i] * value[i];
    }
    store_some<E>((T *)a.dgate + m * a.ldd + n, some, g);
    store_some<E>((T *)a.dup + m * a.ldd + n, some, u);
}

// Rows of `bytes` bytes, `from` bytes apart, to rows `to` bytes apart, 16 bytes to a thread; `to` is a multiple of 16, the rest of a row becomes zero.
template <int BYTES>
__global__ __launch_bounds__(256) void move_rows_kernel(const char *in, char *out, long rows, long bytes, long from, long to) {
    const long across = to / 16, id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= across * rows) return;
    const long m = id / across, c = 16 * (id - m * across);
    *reinterpret_cast<u32x4 *>(out + m * to + c) = load_guarded<BYTES>(in + m * from + c, bytes - c);
}

}  // namespace tops
#endif
