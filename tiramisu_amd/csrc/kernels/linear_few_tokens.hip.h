// The products of linear_tiles.hip.h for few rows of x (one token of each of up to 64 sequences): bound by the bytes of the weights, which
// are read once, straight into registers in the matrix instruction's layout.
// A workgroup computes 16 columns of C (GATED: of gate and of up) for all rows: 16 rows of the weights against up to TILES x 16 rows of x with
// v_mfma_f32_16x16x32, the weights as the instruction's rows.  k is dealt to the wavefronts in units of 128 bytes of a row (every
// line of the weights is read by one wavefront, by two loads that follow each other), up to BATCH units of loads are in flight in each (one token, 4096 x 4096:
// with 8 units 8.1 us, 5.4 TB/s behind the launch; with 4 8.7), and the wavefronts' sums are added through LDS.  x is read by every workgroup, from the L2; rows behind the last read the last one again.
// Addresses may be any multiple of an element.
#ifndef TIRAMISU_AMD_LINEAR_FEW_TOKENS_HIP_H
#define TIRAMISU_AMD_LINEAR_FEW_TOKENS_HIP_H
#include "linear_tiles.hip.h"

namespace tops {

constexpr int FEW_WAVES = 8, FEW_ROWS = 16;
constexpr int few_lds_bytes(int tiles, bool gated) { return FEW_WAVES * (gated ? 2 : 1) * tiles * 1024; }

template <int E>
__device__ __forceinline__ f32x4 multiply_16(u32x4 rows, u32x4 columns, f32x4 c) {
    if constexpr (E == F8) {
        const long a0 = (long)(((uint64_t)rows[1] << 32) | rows[0]), a1 = (long)(((uint64_t)rows[3] << 32) | rows[2]);
        const long b0 = (long)(((uint64_t)columns[1] << 32) | columns[0]), b1 = (long)(((uint64_t)columns[3] << 32) | columns[2]);
        c = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(a0, b0, c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(a1, b1, c, 0, 0, 0);
    } else if constexpr (E == BF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, rows), __builtin_bit_cast(bf16x8, columns), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, rows), __builtin_bit_cast(f16x8, columns), c, 0, 0, 0);
    }
}

template <int E, int Y, int EPILOGUE, int TILES>
__global__ __launch_bounds__(64 * FEW_WAVES) void few_tokens_kernel(product_arguments p) {
    constexpr int BYTES = E == F8 ? 1 : 2, PARTS = EPILOGUE == GATED ? 2 : 1, BATCH = TILES * PARTS >= 4 ? 2 : TILES * PARTS == 2 ? 4 : 8;
    extern __shared__ __attribute__((aligned(16))) char shared_bytes[];
    __attribute__((address_space(3))) f32x4 *const sums = (__attribute__((address_space(3))) f32x4 *)shared_bytes;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, group = lane >> 4;
    const long n0 = (long)blockIdx.x * FEW_ROWS, bytes = (long)p.K * BYTES;

    const char *w[PARTS], *x[TILES];
    const long weight_row = min(n0 + l16, (long)p.N - 1);
    w[0] = (const char *)p.b + weight_row * p.ldb * BYTES + 16 * group;
    if constexpr (PARTS == 2) w[1] = (const char *)p.b2 + weight_row * p.ldb2 * BYTES + 16 * group;
#pragma unroll
    for (int i = 0; i < TILES; i++) x[i] = (const char *)p.a + (long)min(16 * i + l16, p.M - 1) * p.lda * BYTES + 16 * group;

    f32x4 acc[PARTS][TILES];
#pragma unroll
    for (int q = 0; q < PARTS; q++)
#pragma unroll
        for (int i = 0; i < TILES; i++) acc[q][i] = f32x4{0.f, 0.f, 0.f, 0.f};

    // what the epilogue of 8 columns of row m reads, ahead of the product
    const int id = threadIdx.x, m = id >> 1, c0 = 8 * (id & 1);
    const long n = n0 + c0;
    const int some = (int)min(8L, p.N - n);
    const bool mine = m < p.M && m < 16 * TILES && some > 0;
    column_pieces pieces;
    u32x4 residual = {0, 0, 0, 0};
    float scale = 1.f;
    if (mine) {
        load_column_pieces(p, pieces, n, some);
        if (EPILOGUE == LINEAR && p.residual) residual = load_guarded<2>((const char *)p.residual + 2 * ((long)m * p.ldr + n), 2 * some);
        if (E == F8) scale = p.a_scale[m];
    }

    const int whole = (int)(bytes / 128), units = (int)((bytes + 127) / 128);
    int u = wave;
    // as many units at a time as are left, by halves
    auto take = [&](auto batch_c) {
        constexpr int B = decltype(batch_c)::value;
        for (; u + (B - 1) * FEW_WAVES < whole; u += B * FEW_WAVES) {
            u32x4 fw[B][2][PARTS], fx[B][2][TILES];
#pragma unroll
            for (int b = 0; b < B; b++)
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const long at = (long)(u + b * FEW_WAVES) * 128 + 64 * half;
#pragma unroll
                    for (int q = 0; q < PARTS; q++) fw[b][half][q] = *reinterpret_cast<const u32x4_any *>(w[q] + at);
#pragma unroll
                    for (int i = 0; i < TILES; i++) fx[b][half][i] = *reinterpret_cast<const u32x4_any *>(x[i] + at);
                }
#pragma unroll
            for (int b = 0; b < B; b++)
#pragma unroll
                for (int half = 0; half < 2; half++)
#pragma unroll
                    for (int q = 0; q < PARTS; q++)
#pragma unroll
                        for (int i = 0; i < TILES; i++) acc[q][i] = multiply_16<E>(fw[b][half][q], fx[b][half][i], acc[q][i]);
        }
    };
    if constexpr (BATCH >= 8) take(std::integral_constant<int, 8>());
    if constexpr (BATCH >= 4) take(std::integral_constant<int, 4>());
    take(std::integral_constant<int, 2>());
    take(std::integral_constant<int, 1>());
    for (; u < units; u += FEW_WAVES) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const long at = (long)u * 128 + 64 * half, left = bytes - at - 16 * group;
            u32x4 fw[PARTS], fx[TILES];
#pragma unroll
            for (int q = 0; q < PARTS; q++) fw[q] = load_guarded<BYTES>(w[q] + at, left);
#pragma unroll
            for (int i = 0; i < TILES; i++) fx[i] = load_guarded<BYTES>(x[i] + at, left);
#pragma unroll
            for (int q = 0; q < PARTS; q++)
#pragma unroll
                for (int i = 0; i < TILES; i++) acc[q][i] = multiply_16<E>(fw[q], fx[i], acc[q][i]);
        }
    }

    // sums[wave][part][tile][lane]: a lane holds rows 4 group .. + 3 of the weights for row l16 of x
#pragma unroll
    for (int q = 0; q < PARTS; q++)
#pragma unroll
        for (int i = 0; i < TILES; i++) sums[((wave * PARTS + q) * TILES + i) * 64 + lane] = acc[q][i];
    __syncthreads();
    if (!mine) return;
    float z[PARTS][8];
#pragma unroll
    for (int q = 0; q < PARTS; q++) {
#pragma unroll
        for (int i = 0; i < 8; i++) z[q][i] = 0.f;
#pragma unroll
        for (int v = 0; v < FEW_WAVES; v++)
#pragma unroll
            for (int four = 0; four < 2; four++) {
                const f32x4 s = sums[((v * PARTS + q) * TILES + (m >> 4)) * 64 + (c0 / 4 + four) * 16 + (m & 15)];
#pragma unroll
                for (int i = 0; i < 4; i++) z[q][4 * four + i] += s[i];
            }
    }
    column_terms columns;
    widen_column_pieces<Y>(p, pieces, columns);
    if constexpr (EPILOGUE == GATED) finish_gated<Y>(p, columns, z[0], z[1], scale, m, n, some);
    else {
        float r[8];
        widen<Y>(residual, r);
        finish_linear<Y>(p, columns, z[0], r, scale, m, n, some);
    }
}

}  // namespace tops
#endif
