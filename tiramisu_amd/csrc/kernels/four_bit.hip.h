// Products with weights in 4 bits: e2m1 values (a sign, two bits of exponent, one of mantissa: 0, 1/2, 1, 3/2, 2, 3, 4, 6), two to a byte with the first in the low half,
// and for each 32 along a row a power of two, as its exponent and 127 (e8m0).  gfx950 converts a pair of values, scaled, to a pair of 16-bit numbers in one
// instruction; a value has two significant bits, so bfloat16 holds every scaled one below 2^128 exactly, down to 2^-128 (which the matrix instruction takes as it is), and
// float16 those within its range; larger ones are infinite.
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

// Few tokens: 16 rows of the weights against up to TILES x 16 of x for every SPLIT of a workgroup's wavefronts, which share their k; the weights are the matrix instruction's
// rows.  x is 4 times the weights' bytes (16 tokens), so it comes into LDS once for all wavefronts, CHUNK elements of every row at a time; weights go from memory straight into registers,
// all of a chunk's at once.
//   * A lane loads 16 bytes of a row, which are 32 weights and one scale's; their eights are the k of four matrix instructions.  A unit is 64 bytes of a
//     row: 128 weights.  Lanes of one k take the 16 bytes 0, 2, 1, 3 of it.
//   * LDS: blocks of 64 k, [16 TILES tokens][8 granules of 16 bytes], granule q of token t at q ^ (t >> 1): with the order above the sixteen lanes that a read serves together meet
//     distinct banks.
// With x read by every wavefront from the caches instead, whose lanes of one instruction touch 64 lines, 16384 x 4096 took 17.3 us for one token and 27.6 for 16; gated 8192 x 2048, 16 tokens,
// 10.8.
constexpr int four_bit_chunk(int tiles) { return 4096 / tiles; }
template <int E, int EPILOGUE, int TILES, int SPLIT>
__global__ __launch_bounds__(64 * FEW_WAVES) void four_bit_few_kernel(four_bit_arguments a) {
    constexpr int PARTS = EPILOGUE == GATED ? 2 : 1, CHUNK = four_bit_chunk(TILES), BLOCK = 16 * TILES * 128, UNITS = (CHUNK / 128 + SPLIT - 1) / SPLIT;
    extern __shared__ __attribute__((aligned(16))) char shared_bytes[];
    lds_char *const lds = (lds_char *)shared_bytes;
    typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
    product_arguments p = a.p;
    const long m0 = (long)blockIdx.y * 16 * TILES;
    p.a = (const char *)p.a + m0 * p.lda * 2;
    if (p.residual) p.residual = (const char *)p.residual + m0 * p.ldr * 2;
    p.y = (char *)p.y + m0 * p.N * 2;
    p.M = p.rows_above = p.split_row = (int)min(p.M - m0, 16L * TILES);
    const int lane = threadIdx.x & 63, w8 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), team = w8 / SPLIT, wave = w8 % SPLIT;
    const int l16 = lane & 15, group = lane >> 4, piece = (group & 1) * 2 + (group >> 1);
    const long n0 = ((long)blockIdx.x * (FEW_WAVES / SPLIT) + team) * FEW_ROWS, bytes = (p.K + 1) / 2;

    const char *w[PARTS];
    const uint8_t *scale[PARTS];
    const long weight_row = min(n0 + l16, (long)p.N - 1);
    w[0] = (const char *)p.b + weight_row * p.ldb + 16 * piece;
    scale[0] = a.scale + weight_row * a.lds;
    if constexpr (PARTS == 2) {
        w[1] = (const char *)p.b2 + weight_row * p.ldb2 + 16 * piece;
        scale[1] = a.scale_2 + weight_row * a.lds_2;
    }
    f32x4 acc[PARTS][TILES];
#pragma unroll
    for (int q = 0; q < PARTS; q++)
#pragma unroll
        for (int i = 0; i < TILES; i++) acc[q][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    // what the epilogue of 8 columns of row m reads, ahead of the product
    const int id = threadIdx.x % (64 * SPLIT), m = id >> 1, c0 = 8 * (id & 1);
    const long n = n0 + c0;
    const int some = (int)min(8L, p.N - n);
    const bool mine = m < p.M && m < 16 * TILES && some > 0;
    column_pieces pieces;
    u32x4 residual = {0, 0, 0, 0};
    if (mine) {
        load_column_pieces(p, pieces, n, some);
        if (EPILOGUE == LINEAR && p.residual) residual = load_guarded<2>((const char *)p.residual + 2 * ((long)m * p.ldr + n), 2 * some);
    }

    // a unit's weights against x's four eights
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
    const long x_bytes = ((p.M - 1L) * p.lda + p.K) * 2;
    const __amdgpu_buffer_rsrc_t x = __builtin_amdgcn_make_buffer_rsrc((void *)p.a, 0, (int)min((x_bytes + 3) & ~3L, 0x7ffffffcL), 0x00020000);
    const int whole = p.K / 128;                                           // units
    for (int first = 0; first < whole; first += CHUNK / 128) {
        const int units = min(CHUNK / 128, whole - first);
        if (first > 0) __syncthreads();                                    // (the chunk before has been read)
        // 8 tokens of a block to an instruction; none where no token of them is there, whose columns nobody stores
        const int eights = (p.M + 7) / 8;
        for (int i = w8; i < units * 2 * eights; i += FEW_WAVES) {
            const int block = i / eights, eight = i - block * eights, token = 8 * eight + lane / 8, q = (lane % 8) ^ ((token >> 1) & 7);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(x, (__attribute__((address_space(3))) void *)(lds + block * BLOCK + eight * 1024), 16,
                                                     (int)(token * p.lda * 2) + (first * 128 + block * 64) * 2 + 16 * q, 0, 0, 0);
        }
        // `each` units next to each other to a wavefront: whole lines of weights, and the scales of four units, four to a unit, in one load
        const int each = (units + SPLIT - 1) / SPLIT, begin = wave * each, own = min(each, units - begin);
        u32x4 fw[UNITS][PARTS], scales[(UNITS + 3) / 4][PARTS];
#pragma unroll
        for (int i = 0; i < UNITS; i++) {
            if (i >= own) break;
            const long u = first + begin + i;
#pragma unroll
            for (int q = 0; q < PARTS; q++) {
                fw[i][q] = *reinterpret_cast<const u32x4_any *>(w[q] + u * 64);
                if (i % 4 == 0) scales[i / 4][q] = load_to_end<4>((const char *)scale[q] + u * 4, 4L * (whole - u), 4L * whole);
            }
        }
        wait_loads<0>();
        __syncthreads();
#pragma unroll
        for (int i = 0; i < UNITS; i++) {
            if (i >= own) break;
            const int u = begin + i;
            uint32_t exponent[PARTS];
#pragma unroll
            for (int q = 0; q < PARTS; q++) exponent[q] = (scales[i / 4][q][i % 4] >> (8 * piece)) & 255;
            u32x4 fx[4][TILES];
#pragma unroll
            for (int step = 0; step < 4; step++)
#pragma unroll
                for (int j = 0; j < TILES; j++) {
                    const int token = 16 * j + l16, q = 4 * (piece & 1) + step;
                    fx[step][j] = *reinterpret_cast<const __attribute__((address_space(3))) u32x4 *>(lds + (2 * u + (piece >> 1)) * BLOCK + (token * 8 + (q ^ ((token >> 1) & 7))) * 16);
                }
            multiply(fw[i], fx, exponent);
        }
    }
    // behind the whole units, from memory
    if (whole * 128 < p.K && wave == whole % SPLIT) {
        const long at = whole * 64L, left = bytes - at - 16 * piece, left_x = 2L * p.K - 4 * at - 64 * piece;
        const int weights = (int)(p.K - 2 * at) - 32 * piece;
        u32x4 fw[PARTS], fx[4][TILES];
        uint32_t exponent[PARTS];
#pragma unroll
        for (int q = 0; q < PARTS; q++) {
            fw[q] = load_to_end<1>(w[q] + at, left, bytes);
            // (of an odd number of weights the last byte's high half is none, whatever it holds: in float16 a large scale would make it infinity, and its product with x's zero NaN)
#pragma unroll
            for (int i = 0; i < 4; i++) fw[q][i] &= weights >= 8 * i + 8 ? 0xffffffffu : weights <= 8 * i ? 0u : (1u << (4 * (weights - 8 * i))) - 1;
            exponent[q] = left > 0 ? scale[q][whole * 4L + piece] : 127;
        }
#pragma unroll
        for (int step = 0; step < 4; step++)
#pragma unroll
            for (int i = 0; i < TILES; i++)
                fx[step][i] = load_to_end<2>((const char *)p.a + (long)min(16 * i + l16, p.M - 1) * p.lda * 2 + 4 * at + 64 * piece + 16 * step, left_x - 16 * step, 2L * p.K);
        multiply(fw, fx, exponent);
    }

    // sums[wave][part][tile][lane]: a lane holds rows 4 group .. + 3 of the weights for row l16 of x
    lds_f32x4 *const sums = (lds_f32x4 *)lds + team * SPLIT * PARTS * TILES * 64;
    __syncthreads();
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
        for (int v = 0; v < SPLIT; v++)
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

// The weights as 16-bit numbers, for many tokens: 8 of a row to a thread, rows `to` elements apart, a multiple of 8 (what is behind the last of a row
// is not a number of its).  Bound by the bytes written: 4096 x 4096 9 us (32 weights to a thread, whose stores are 64 bytes apart, 16).
template <int E>
__global__ __launch_bounds__(256) void widen_rows_kernel(const char *q, const uint8_t *scale, long ldq, long lds, long rows, long columns, char *out, long to) {
    const long across = to / 8, id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= across * rows) return;
    const long r = id / across, c = id - r * across, bytes = (columns + 1) / 2;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (4 * c + i < bytes) word |= (uint32_t)(uint8_t)q[r * ldq + 4 * c + i] << (8 * i);
    *reinterpret_cast<u32x4 *>(out + (r * to + 8 * c) * 2) = widen_8<E>(word, scale_of(scale[r * lds + c / (GROUP / 8)]));
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
