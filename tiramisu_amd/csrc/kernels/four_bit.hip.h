// Products with weights in 4 bits: e2m1 values (a sign, two bits of exponent, one of mantissa: 0, 1/2, 1, 3/2, 2, 3, 4, 6), two to a byte with the first in the low half,
// and for each 32 along a row a power of two, as its exponent and 127 (e8m0).  gfx950 converts a pair of values, scaled, to a pair of 16-bit numbers in one
// instruction; a value has two significant bits, so bfloat16 holds every scaled one exactly, and float16 those within its range.
#ifndef TIRAMISU_AMD_FOUR_BIT_HIP_H
#define TIRAMISU_AMD_FOUR_BIT_HIP_H
#include "linear_few_tokens.hip.h"

namespace tfour {

using namespace tops;

constexpr int GROUP = 32;                   // weights of a row with one scale
constexpr float E2M1_MOST = 6.f;

struct four_bit_arguments {
    product_arguments p;                    // b, b2: the values; ldb, ldb2: bytes from row to row
    const uint8_t *scale, *scale_2;
    long lds, lds_2;                        // bytes from row to row of the scales
};

// The number that an exponent byte stands for: 255 is NaN
__device__ __forceinline__ float scale_of(uint32_t byte) { return byte == 255 ? __builtin_nanf("") : byte == 0 ? 0x1p-127f : __builtin_bit_cast(float, byte << 23); }

// Eight values of a word, scaled
template <int E>
__device__ __forceinline__ u32x4 widen_8(uint32_t word, float scale) {
    u32x4 w;
    if constexpr (E == BF16) {
        w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 0));
        w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 1));
        w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 2));
        w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, 3));
    } else {
        w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 0));
        w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 1));
        w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 2));
        w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, 3));
    }
    return w;
}

// Few tokens: as linear_few_tokens.hip.h, with 16 rows of the weights against up to TILES x 16 of x in a workgroup.  A lane loads 16 bytes of a row, which are 32
// weights and one scale's; their eights are the k of four matrix instructions, whose lanes of x hold the same k.  A unit, dealt to the wavefronts in turn, is 128
// bytes of a row: 256 weights in two loads.
template <int E, int EPILOGUE, int TILES>
__global__ __launch_bounds__(64 * FEW_WAVES) void four_bit_few_kernel(four_bit_arguments a) {
    constexpr int PARTS = EPILOGUE == GATED ? 2 : 1, BATCH = TILES * PARTS > 1 ? 1 : 2;
    extern __shared__ __attribute__((aligned(16))) char shared_bytes[];
    __attribute__((address_space(3))) f32x4 *const sums = (__attribute__((address_space(3))) f32x4 *)shared_bytes;
    product_arguments p = a.p;
    const long m0 = (long)blockIdx.y * 16 * TILES;
    p.a = (const char *)p.a + m0 * p.lda * 2;
    if (p.residual) p.residual = (const char *)p.residual + m0 * p.ldr * 2;
    p.y = (char *)p.y + m0 * p.N * 2;
    if (p.pre) p.pre = (char *)p.pre + m0 * p.N * 2;
    if (p.pre2) p.pre2 = (char *)p.pre2 + m0 * p.N * 2;
    p.M = p.rows_above = p.split_row = (int)min(p.M - m0, 16L * TILES);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, group = lane >> 4;
    const long n0 = (long)blockIdx.x * FEW_ROWS, bytes = (p.K + 1) / 2;

    const char *w[PARTS], *x[TILES];
    const uint8_t *scale[PARTS];
    const long weight_row = min(n0 + l16, (long)p.N - 1);
    w[0] = (const char *)p.b + weight_row * p.ldb + 16 * group;
    scale[0] = a.scale + weight_row * a.lds + group;
    if constexpr (PARTS == 2) {
        w[1] = (const char *)p.b2 + weight_row * p.ldb2 + 16 * group;
        scale[1] = a.scale_2 + weight_row * a.lds_2 + group;
    }
    bool token[TILES];
#pragma unroll
    for (int i = 0; i < TILES; i++) {
        token[i] = 16 * i + l16 < p.M;
        x[i] = (const char *)p.a + (long)min(16 * i + l16, p.M - 1) * p.lda * 2 + 64 * group;
    }

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
    if (mine) {
        load_column_pieces(p, pieces, n, some);
        if (EPILOGUE == LINEAR && p.residual) residual = load_guarded<2>((const char *)p.residual + 2 * ((long)m * p.ldr + n), 2 * some);
    }

    // 64 bytes of a row, 16 of a lane: 32 k
    auto multiply = [&](const u32x4 (&fw)[PARTS], const u32x4 (&fx)[4][TILES], const uint32_t (&exponent)[PARTS]) {
#pragma unroll
        for (int q = 0; q < PARTS; q++) {
            const float s = scale_of(exponent[q]);
#pragma unroll
            for (int step = 0; step < 4; step++) {
                const u32x4 rows = widen_8<E>(fw[q][step], s);
#pragma unroll
                for (int i = 0; i < TILES; i++) acc[q][i] = multiply_16<E>(rows, fx[step][i], acc[q][i]);
            }
        }
    };
    const int whole = (int)(p.K / 256), units = (int)((p.K + 255) / 256);
    int u = wave;
    auto take = [&](auto batch_c) {
        constexpr int B = 2 * decltype(batch_c)::value;
        for (; u + (B / 2 - 1) * FEW_WAVES < whole; u += B / 2 * FEW_WAVES) {
            u32x4 fw[B][PARTS], fx[B][4][TILES];
            uint32_t exponent[B][PARTS];
#pragma unroll
            for (int b = 0; b < B; b++) {
                const long at = (long)(u + b / 2 * FEW_WAVES) * 128 + 64 * (b % 2);
#pragma unroll
                for (int q = 0; q < PARTS; q++) {
                    fw[b][q] = *reinterpret_cast<const u32x4_any *>(w[q] + at);
                    exponent[b][q] = scale[q][at / 16];
                }
            }
#pragma unroll
            for (int b = 0; b < B; b++) {
                const long at = (long)(u + b / 2 * FEW_WAVES) * 128 + 64 * (b % 2);
#pragma unroll
                for (int i = 0; i < TILES; i++)
#pragma unroll
                    for (int step = 0; step < 4; step++) {
                        fx[b][step][i] = u32x4{0, 0, 0, 0};
                        if (token[i]) fx[b][step][i] = *reinterpret_cast<const u32x4_any *>(x[i] + 4 * at + 16 * step);
                    }
            }
#pragma unroll
            for (int b = 0; b < B; b++) multiply(fw[b], fx[b], exponent[b]);
        }
    };
    if constexpr (BATCH >= 2) take(std::integral_constant<int, 2>());
    take(std::integral_constant<int, 1>());
    for (; u < units; u += FEW_WAVES) {
#pragma unroll 1
        for (int half = 0; half < 2; half++) {
            const long at = (long)u * 128 + 64 * half, left = bytes - at - 16 * group, left_x = 2L * p.K - 4 * at - 64 * group;
            u32x4 fw[PARTS], fx[4][TILES];
            uint32_t exponent[PARTS];
#pragma unroll
            for (int q = 0; q < PARTS; q++) {
                fw[q] = load_to_end<1>(w[q] + at, left, bytes);
                exponent[q] = left > 0 ? scale[q][at / 16] : 127;
            }
#pragma unroll
            for (int step = 0; step < 4; step++)
#pragma unroll
                for (int i = 0; i < TILES; i++) fx[step][i] = load_to_end<2>(x[i] + 4 * at + 16 * step, left_x - 16 * step, 2L * p.K);
            multiply(fw, fx, exponent);
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
    widen_column_pieces<E>(p, pieces, columns);
    if constexpr (EPILOGUE == GATED) finish_gated<E>(p, columns, z[0], z[1], 1.f, m, n, some);
    else {
        float r[8];
        widen<E>(residual, r);
        finish_linear<E>(p, columns, z[0], r, 1.f, m, n, some);
    }
}

// The weights as 16-bit numbers, for many tokens: 32 of a row to a thread, rows `to` elements apart, a multiple of 8 (what is behind the last of a row
// is not a number of its).
// (16 bytes in, 64 out; bound by the bytes written)
template <int E>
__global__ __launch_bounds__(256) void widen_rows_kernel(const char *q, const uint8_t *scale, long ldq, long lds, long rows, long columns, char *out, long to) {
    const long across = (columns + GROUP - 1) / GROUP, id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= across * rows) return;
    const long r = id / across, g = id - r * across, some = min((long)GROUP, columns - g * GROUP);
    const u32x4 w = load_guarded<1>(q + r * ldq + 16 * g, (some + 1) / 2);
    const float s = scale_of(scale[r * lds + g]);
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (8 * i < some)
            *reinterpret_cast<u32x4 *>(out + (r * to + g * GROUP + 8 * i) * 2) = widen_8<E>(w[i], s);
}

// Rows to 4 bits: scale the smallest power of two by which the group's largest is at most 6 (1 for a group of zeros), values to the nearest, ties to even, of the
// group ahead of any rounding.  One group to a thread.
template <int E>
__global__ __launch_bounds__(256) void quantize_groups_kernel(const void *x, long ld, long rows, long columns, char *q, uint8_t *scale) {
    const long across = (columns + GROUP - 1) / GROUP, id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= across * rows) return;
    const long r = id / across, g = id - r * across;
    const int some = (int)min((long)GROUP, columns - g * GROUP);
    const stored<E> *const from = (const stored<E> *)x + r * ld + g * GROUP;
    float v[GROUP], most = 0.f;
    bool whole = true;
#pragma unroll
    for (int i = 0; i < GROUP; i++) {
        v[i] = i < some ? load_one<E>(from + i) : 0.f;
        most = fmaxf(most, fabsf(v[i]));
        whole = whole && fabsf(v[i]) < __builtin_inff();
    }
    // most <= 6 2^e: with most = f 2^b, 1/2 <= f < 1, that is b - 2 for f up to 3/4, b - 3 for none (6 = 3/4 2^3)
    int b = 0;
    const float f = most > 0.f ? frexpf(most, &b) : 0.f;
    const int e = most > 0.f ? max(-127, b - 3 + (f > 0.75f)) : 0;
    uint32_t words[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < GROUP; i++) {
        const float a = ldexpf(fabsf(v[i]), -e);
        // middles between the values; a tie goes to the even code
        uint32_t code = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) + (a >= 3.5f) + (a > 5.f);
        if (__builtin_bit_cast(uint32_t, v[i]) >> 31) code |= 8;
        words[i / 8] |= code << (4 * (i % 8));
    }
    const long bytes = (columns + 1) / 2;
    char *const to = q + r * bytes + 16 * g;
    for (int i = 0; i < (some + 1) / 2; i++) to[i] = (char)(words[i / 4] >> (8 * (i % 4)));
    scale[r * across + g] = whole ? (uint8_t)(e + 127) : 255;
}

}  // namespace tfour
#endif
