// Matrix products of the transformer operators on tiles: C[m, n] = sum_k A(m, k) B(n, k) with fp32 accumulation on the matrix cores, and
// the operator's epilogue on the accumulators.  Each operand lies either with k along its rows ([m][k], what x and weights
// are in a forward pass) or with k down its columns ([k][m], what weights are for the gradient of the input, and both operands for
// the gradient of the weights); 16-bit elements either way, 8-bit ones (e4m3) with k along the rows.
//
// Slices of 128 bytes of k a row go from memory straight into an LDS ring (buffer loads with LDS as their destination, 16 bytes a lane):
//   * k along the rows: [rows][8 granules of 16 bytes], granule q of row m at q ^ swizzle(m); one 16-byte read is a lane's eight k.
//   * k down the columns: [64 k][rows / 8 granules], granule g of row k at g ^ swizzle(k); two transposing reads
//     (ds_read_b64_tr_b16) are a lane's eight k: within 16 lanes, lane L receives element L % 4 of the 8 bytes that lanes L / 4 + 4 i address.
// Both keep reads and loads free of bank conflicts (swizzles as in gemm_mfma_bf16.hip.h).  One barrier a slice retires its stage and
// publishes the next; the instruction order is pinned so that fragments are read a whole step of matrix instructions ahead.
//
// Nothing outside the operands is read: descriptors begin at the tile and end with the operand, so rows behind the last read as zero; k behind the last
// is set to zero in registers where k runs along the rows (the row goes on into the next one there, whose infinities must not meet a zero of
// the other operand), and is behind the descriptor's end where it runs down the columns.
// The descriptor of an operand with k down its columns moves on with the slices, so operands may be larger than 4 GiB.
//
// 8-bit products: the matrix instructions (all that gfx950 has for e4m3) add eight neighbouring products at a time, each cut off below 2^-12 of the
// largest one's power of two, and accumulate these sums in fp32.  Operands of 4 significant bits lose little by it (the result of a
// 4096-long product of normal numbers is as close to 64 bits as without, at bf16's rounding); converting them to bf16 first would halve the rate.
//
// The matrix instruction takes B's rows as its rows, so that a lane's accumulator registers run along a row of C: four 16-byte LDS
// stores a 32 x 32 block turn a strip of 32 rows of a wavefront into rows of 8 columns a lane, and bias, residual and outputs
// are read and written in 16-byte pieces, whole lines at a time.
//
// What it reaches, and what holds it: bf16 4096^3 98 - 102 us, 1350 - 1400 TFLOP/s (on zeros 82 us: the power that random bits draw); gated 4096 x 8192 x
// 4096 with both projections kept 420 - 440 us, 1250 - 1310; e4m3 4096^3 62 - 69 us, 2000 - 2200 TFLOP/s, matrix cores busy 45 % of the time: slices come
// into a compute unit's LDS at about 40 bytes a nanosecond, and 256 x 256 is the largest tile whose sums fit the registers.  Slices of 64 bytes in a
// deeper ring are no faster (bf16 103 us, e4m3 64), nor are rows padded to other strides.  Small products are one round of tiles: launch, first slices and
// epilogue stand one after the other (2000 x 1500 x 1000 f16 17.3 us a call with gelu and the sums kept, 16.3 with gelu, 14.7 without).
#ifndef TIRAMISU_AMD_LINEAR_TILES_HIP_H
#define TIRAMISU_AMD_LINEAR_TILES_HIP_H
#include <type_traits>

#include "operator_elements.hip.h"

namespace tops {

// What an epilogue does.  LINEAR: z = sum [a_scale b_scale] + bias; pre = z; y = activation(z) + residual.  GATED: half of the tile's columns are
// gate, half up (rows n of b and of b2): h = activation(gate) up, and both where kept.
enum epilogue : int { LINEAR = 0, GATED = 1 };

struct product_arguments {
    const void *a, *b, *b2;                 // b2: GATED, the second weight
    const void *a_more, *b_more;            // a second pair of operands added to the product (null: none), of the same sizes and strides
    long lda, ldb, ldb2, ldb_more;          // elements
    int M, N, K;                            // N: columns of C (GATED: of h)
    const void *bias, *residual;
    const float *a_scale, *b_scale, *b2_scale;
    long ldr;
    void *y, *pre, *pre2;                   // dense, rows of N
    void *y_below;                          // rows from `split_row` on go here (row split_row first); rows from `rows_above` to it nowhere
    int split_row, rows_above;
    int activation;
    float *partial;                         // sums only, [split][M][N] (GATED: [split][2][M][N]); null: the whole product in one workgroup
    int slices_per_split;
};

template <int E_, int BM_, int BN_, int WGM_, int WGN_, int STAGES_, bool A_ROWS_, bool B_ROWS_, int EPILOGUE_, int F_>
struct tile_config {
    static constexpr int F = F_;                                           // rows of a fragment: matrix instructions of F x F
    static constexpr int E = E_, BM = BM_, BN = BN_, WGM = WGM_, WGN = WGN_, STAGES = STAGES_, EPILOGUE = EPILOGUE_;
    static constexpr bool A_ROWS = A_ROWS_, B_ROWS = B_ROWS_;              // k along the rows
    static constexpr int BYTES = E == F8 ? 1 : 2, BK = 128 / BYTES;
    static constexpr int NW = WGM * WGN, NT = 64 * NW;
    static constexpr int WM = BM / WGM, WN = BN / WGN, TM = WM / F, TN = WN / F;
    static constexpr int STEP = F == 16 ? (E == F8 ? 128 : 64) : (E == F8 ? 64 : 32);     // bytes of a row in a matrix step
    static constexpr int A_STAGE = BM * 128, B_STAGE = BN * 128, STAGE = A_STAGE + B_STAGE;
    static constexpr int LA = BM / 8 / NW, LB = BN / 8 / NW;               // loads of a wavefront for a slice
    static constexpr int STRIP = WN + 4;                                   // floats of a row in the epilogue's strip: 16-byte stores of 16 rows fill the banks
    static constexpr int EPILOGUE_BYTES = NW * 32 * STRIP * 4;
    static constexpr int LDS_BYTES = STAGES * STAGE > EPILOGUE_BYTES ? STAGES * STAGE : EPILOGUE_BYTES;
    static constexpr int COLUMNS = EPILOGUE == GATED ? BN / 2 : BN;        // of C
    static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "slices split evenly over the wavefronts");
    static_assert(E != F8 || (A_ROWS && B_ROWS), "8-bit operands have k along their rows");
    static_assert(EPILOGUE != GATED || (TN % 2 == 0 && BN % 128 == 0 && B_ROWS), "a wavefront holds gate and up of the same columns");
    static_assert(LDS_BYTES <= 160 * 1024, "LDS of a compute unit");
};

template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

typedef __attribute__((address_space(3))) char lds_char;

// An operand's slices: what a lane loads, and where.
template <int BYTES, int ROWS, bool K_ALONG_ROWS, int LOADS, int F>
struct operand_loader {
    static constexpr int G = K_ALONG_ROWS ? 8 : ROWS / 8;                  // granules of a row in LDS
    // Lanes that an LDS read serves together meet distinct banks: of a 16-byte read they are 16 at a time, 0-3, 12-15, 20-23 and 24-27 the first of
    // them, whose rows and granules F and the element's size decide (with the first form for all, 16-bit fragments of 16 rows took two cycles for
    // one: half of the LDS's busy cycles); of a transposing one 16 or 32.
    static __device__ __forceinline__ int swizzle(int row) {
        if (K_ALONG_ROWS) return (F == 16 && BYTES == 2 ? row >> 1 : row ^ (row >> 3)) & 7;
        const int eighth = F == 16 ? (row >> 3) & 1 : 0;                   // (F == 16: such 32 lanes read k and k + 8)
        return G == 8 ? 2 * ((row & 3) ^ eighth) : (((row & 1) << 2) | ((row & 2) ? 10 : 0)) ^ (eighth << 1);
    }
    const char *base;
    long left, step;                        // bytes from base to the operand's end; from slice to slice (k down the columns)
    int offset[LOADS], along;               // per lane; bytes of k requested so far (k along the rows)

    // `first`: the tile's first row; `rows`, `k`: of the operand, from element k0 on
    __device__ __forceinline__ void start(const void *p, long ld, long first, long rows, long k0, long k, int wave, int lane) {
        const char *b = (const char *)p;
        if (K_ALONG_ROWS) {
            base = b + (first * ld + k0) * BYTES;
            left = ((rows - 1 - first) * ld + k) * BYTES;
            step = 0;
        } else {
            base = b + (k0 * ld + first) * BYTES;
            left = ((k - 1) * ld + (rows - first)) * BYTES;
            step = 64 * ld * BYTES;
        }
        along = 0;
#pragma unroll
        for (int v = 0; v < LOADS; v++) {
            const int g = (wave * LOADS + v) * 64 + lane, row = g / G, q = (g % G) ^ swizzle(row);
            offset[v] = (int)(row * ld * BYTES) + q * 16;
        }
    }
    // (a dword that begins inside an operand and ends outside reads as zero: the end is moved to a whole one)
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t descriptor() const {
        const long n = (left + 3) & ~3L;
        return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, n > 0x7ffffffcL ? 0x7ffffffc : n < 0 ? 0 : (int)n, 0x00020000);
    }
    __device__ __forceinline__ void load(lds_char *stage, int wave, int v) const {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(descriptor(), (__attribute__((address_space(3))) void *)(stage + (wave * LOADS + v) * 1024), 16, offset[v], along, 0, 0);
    }
    __device__ __forceinline__ void advance() {
        if (K_ALONG_ROWS) along += 128;
        else { base += step; left -= step; }
    }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef int s32x4 __attribute__((ext_vector_type(4)));
typedef int s32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// A lane's share of F rows of an operand for one matrix step: 8 k of 16 bits, or 32 of 8 bits.
template <int E, bool K_ALONG_ROWS> struct fragment {
    u32x4 w[E == F8 ? 2 : 1];
    s16x4 half[2];                          // (k down the columns: as the transposing reads give them)
};
template <int F> struct block_sums;         // a lane's share of the sums of F x F
template <> struct block_sums<16> { typedef f32x4 type; };
template <> struct block_sums<32> { typedef f32x16 type; };

// The 16 bytes of k of a matrix step that piece `part` of a lane's fragment holds: their granule within a slice.
template <int E, int F>
__device__ __forceinline__ int granule_of(int step, int part, int lane) {
    const int group = lane / F, groups = 64 / F;
    return E == F8 ? 2 * (groups * step + group) + part : groups * step + group;
}
// One LDS read of the fragment of the F rows from `row` on of the slice at `s`, step `step`; L: the operand's loader.
template <class L, int F, int E>
__device__ __forceinline__ void read_piece(fragment<E, true> &f, lds_char *s, int row, int step, int part, int lane) {
    const int m = row + lane % F, q = granule_of<E, F>(step, part, lane);
    f.w[part] = *reinterpret_cast<const __attribute__((address_space(3))) u32x4 *>(s + (m * 8 + (q ^ L::swizzle(m))) * 16);
}
template <class L, int F, int E>
__device__ __forceinline__ void read_piece(fragment<E, false> &f, lds_char *s, int row, int step, int part, int lane) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const int l16 = lane & 15, group = lane >> 4;
    const int k = F == 16 ? 32 * step + 8 * group + (l16 >> 2) + 4 * part : 16 * step + 8 * (group >> 1) + (l16 >> 2) + 4 * part;
    const int m = row + (F == 16 ? 0 : 16 * (group & 1)) + 4 * (l16 & 3);
    f.half[part] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(s + (k * L::G + ((m >> 3) ^ L::swizzle(k))) * 16 + (m & 7) * 2));
}

// (16 x 16 blocks take less power than 32 x 32 ones on operands of random bits: from registers 2030 and 1800 TFLOP/s of bf16, 4350 and 4000 of e4m3;
// on zeros, where power does not limit, 2430 and 2450, 4970 and 4970)
template <int E, bool AR, bool BR, class S>
__device__ __forceinline__ S multiply(const fragment<E, AR> &rows, const fragment<E, BR> &columns, S c) {
    constexpr bool SMALL = sizeof(S) == 16;
    if constexpr (E == F8) {
        const s32x8 a = __builtin_shufflevector(__builtin_bit_cast(s32x4, rows.w[0]), __builtin_bit_cast(s32x4, rows.w[1]), 0, 1, 2, 3, 4, 5, 6, 7);
        const s32x8 b = __builtin_shufflevector(__builtin_bit_cast(s32x4, columns.w[0]), __builtin_bit_cast(s32x4, columns.w[1]), 0, 1, 2, 3, 4, 5, 6, 7);
        if constexpr (SMALL) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
        else return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
    } else {
        s16x8 a, b;
        if constexpr (AR) a = __builtin_bit_cast(s16x8, rows.w[0]); else a = __builtin_shufflevector(rows.half[0], rows.half[1], 0, 1, 2, 3, 4, 5, 6, 7);
        if constexpr (BR) b = __builtin_bit_cast(s16x8, columns.w[0]); else b = __builtin_shufflevector(columns.half[0], columns.half[1], 0, 1, 2, 3, 4, 5, 6, 7);
        if constexpr (E == BF16 && SMALL) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
        else if constexpr (E == BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
        else if constexpr (SMALL) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
}

// Adds the product of one pair of operands' rows from m0 and n0, K elements of k, to the accumulators.  b, b2: B's operand (GATED: gate and up).
// (The operands are __restrict__ so that the compiler does not take a transposing read of LDS for one that may see a load still on its way there: it
// waited for every load ahead of each of them, 205 us where 105 are enough.)
template <class C>
__device__ __forceinline__ void accumulate(typename block_sums<C::F>::type (&acc)[C::TM][C::TN], const void *__restrict__ a, long lda, const void *__restrict__ b, long ldb, const void *__restrict__ b2, long ldb2, long M, long N,
                                           long m0, long n0, long k0, long K, lds_char *lds) {
    constexpr int TM = C::TM, TN = C::TN, ST = C::STAGES, E = C::E;
    constexpr int F = C::F, Q = 128 / C::STEP;                             // matrix steps of a slice
    constexpr int HALVES = C::EPILOGUE == GATED ? 2 : 1;
    constexpr int LB1 = C::LB / HALVES;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = wave / C::WGN, wn = wave % C::WGN;
    static_assert(C::LB % HALVES == 0, "gate and up are loaded by the same wavefronts");

    operand_loader<C::BYTES, C::BM, C::A_ROWS, C::LA, F> la;
    // (GATED: rows of gate in the first half of B's stage, rows of up in the second)
    operand_loader<C::BYTES, C::BN / HALVES, C::B_ROWS, LB1, F> lb[HALVES];
    la.start(a, lda, m0, M, k0, K, wave, lane);
    lb[0].start(b, ldb, n0, N, k0, K, wave, lane);
    if constexpr (HALVES == 2) lb[1].start(b2, ldb2, n0, N, k0, K, wave, lane);

    auto issue_one = [&](int stage, int v) {
        lds_char *const s = lds + stage * C::STAGE;
        if (v < C::LA) la.load(s, wave, v);
        else if (HALVES == 1 || v < C::LA + LB1) lb[0].load(s + C::A_STAGE, wave, v - C::LA);
        else lb[HALVES - 1].load(s + C::A_STAGE + C::B_STAGE / 2, wave, v - C::LA - LB1);
        if (v == C::LA + C::LB - 1) {
            la.advance();
            lb[0].advance();
            if constexpr (HALVES == 2) lb[1].advance();
        }
    };

    fragment<E, C::A_ROWS> fa[2][TM];
    fragment<E, C::B_ROWS> fb[2][TN];
    constexpr int RA = C::A_ROWS ? (E == F8 ? 2 : 1) : 2, RB = C::B_ROWS ? (E == F8 ? 2 : 1) : 2;      // reads of a fragment
    constexpr int READS = TM * RA + TN * RB, MFMAS = TM * TN;
    // rows of B's stage that fragment j of the wavefront holds (GATED: the first half of the fragments gate, the others up, of the same columns)
    auto row_of = [&](int j) {
        if (HALVES == 1) return wn * C::WN + j * F;
        constexpr int HALF = HALVES == 2 ? TN / 2 : 1;
        return (j >= HALF ? C::BN / 2 : 0) + wn * (C::WN / 2) + (j % HALF) * F;
    };
    // read r of a step, in the order in which the matrix instructions need them: A's first rows, all of B, the other rows of A
    auto read_one = [&](int stage, int step, int buf, int r) {
        lds_char *const s = lds + stage * C::STAGE;
        if (r < RA || r >= RA + TN * RB) {
            const int i = r < RA ? 0 : 1 + (r - RA - TN * RB) / RA, part = r < RA ? r : (r - RA - TN * RB) % RA;
            read_piece<decltype(la), F>(fa[buf][i], s, wm * C::WM + i * F, step, part, lane);
        } else {
            const int j = (r - RA) / RB, part = (r - RA) % RB;
            // (GATED: the two halves are one block of rows, and the swizzle repeats every 64 of them)
            read_piece<typename std::remove_reference<decltype(lb[0])>::type, F>(fb[buf][j], s + C::A_STAGE, row_of(j), step, part, lane);
        }
    };
    // the last slice: k behind the last is zero in both operands
    auto clear_behind = [&](auto &f, int left, int step) {                // left: bytes of k from the slice's first on
#pragma unroll
        for (int part = 0; part < (E == F8 ? 2 : 1); part++) {
            const int rest = left - 16 * granule_of<E, F>(step, part, lane);
#pragma unroll
            for (int w = 0; w < 4; w++) f.w[part][w] &= rest >= 4 * w + 4 ? 0xffffffffu : rest <= 4 * w ? 0u : (1u << (8 * (rest - 4 * w))) - 1u;
        }
    };
    auto mfma_one = [&](int buf, int idx) {
        const int i = idx / TN, j = idx % TN;
        acc[i][j] = multiply<E, C::B_ROWS, C::A_ROWS>(fb[buf][j], fa[buf][i], acc[i][j]);
    };

    const int KT = (int)((K + C::BK - 1) / C::BK);
    if (KT <= 0) return;
    const int tail = (int)(K - (long)(KT - 1) * C::BK) * C::BYTES;        // bytes of k in the last slice
    constexpr int PER = C::LA + C::LB;
    constexpr int PRE = MFMAS >= 32 ? 8 : MFMAS >= 16 ? 4 : MFMAS > 1 ? 1 : 0;              // matrix instructions of a slice's last step ahead of the barrier
    static_assert((ST - 1) * PER <= 63, "the load counter holds 63");
#pragma unroll
    for (int p = 0; p < ST; p++)
        if (p < KT) {
#pragma unroll
            for (int v = 0; v < PER; v++) issue_one(p, v);
        }
    if (KT >= ST) wait_loads<(ST - 1) * PER>(); else wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int r = 0; r < READS; r++) read_one(0, 0, 0, r);
    // (`first`: which of the two sets of fragments holds the slice's first step)
    auto slice = [&](int stage, int next, auto issue_c, auto more_c, auto first_c) {
        constexpr bool ISSUE = decltype(issue_c)::value, MORE = decltype(more_c)::value;
#pragma unroll
        for (int q = 0; q < Q; q++) {
            const int buf = (q + decltype(first_c)::value) & 1;
            if (!MORE && tail != 128) {
                if constexpr (C::A_ROWS) {
#pragma unroll
                    for (int i = 0; i < TM; i++) clear_behind(fa[buf][i], tail, q);
                }
                if constexpr (C::B_ROWS) {
#pragma unroll
                    for (int j = 0; j < TN; j++) clear_behind(fb[buf][j], tail, q);
                }
            }
            if (q + 1 < Q) {
#pragma unroll
                for (int idx = 0; idx < MFMAS; idx++) {
                    mfma_one(buf, idx);
#pragma unroll
                    for (int r = idx * READS / MFMAS; r < (idx + 1) * READS / MFMAS; r++) read_one(stage, q + 1, buf ^ 1, r);
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else if (MORE) {
#pragma unroll
                for (int idx = 0; idx < PRE; idx++) {
                    mfma_one(buf, idx);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (ISSUE) wait_loads<(ST - 2) * PER>(); else wait_loads<0>();
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int idx = PRE; idx < MFMAS; idx++) {
                    mfma_one(buf, idx);
#pragma unroll
                    for (int r = (idx - PRE) * READS / (MFMAS - PRE); r < (idx - PRE + 1) * READS / (MFMAS - PRE); r++) read_one(next, 0, buf ^ 1, r);
                    if (ISSUE) {
#pragma unroll
                        for (int v = (idx - PRE) * PER / (MFMAS - PRE); v < (idx - PRE + 1) * PER / (MFMAS - PRE); v++) issue_one(stage, v);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            } else {
#pragma unroll
                for (int idx = 0; idx < MFMAS; idx++) mfma_one(buf, idx);
            }
        }
    };
    int kt = 0, stage = 0;
    auto advance = [&]() { kt++; stage = stage + 1 == ST ? 0 : stage + 1; };
    auto following = [&]() { return stage + 1 == ST ? 0 : stage + 1; };
    constexpr auto set_0 = std::integral_constant<int, 0>();
    if constexpr (Q % 2 == 0) {
        for (; kt + ST < KT; advance()) slice(stage, following(), std::true_type(), std::true_type(), set_0);
        for (; kt + 1 < KT; advance()) slice(stage, following(), std::false_type(), std::true_type(), set_0);
    } else {
        // one step a slice: slices alternate between the sets, two to a turn of the loop; the last few move theirs back
        constexpr auto set_1 = std::integral_constant<int, 1>();
        auto move_back = [&]() {
#pragma unroll
            for (int i = 0; i < TM; i++) fa[0][i] = fa[1][i];
#pragma unroll
            for (int j = 0; j < TN; j++) fb[0][j] = fb[1][j];
        };
        while (kt + ST + 1 < KT) {
            slice(stage, following(), std::true_type(), std::true_type(), set_0);
            advance();
            slice(stage, following(), std::true_type(), std::true_type(), set_1);
            advance();
        }
        for (; kt + ST < KT; advance()) { slice(stage, following(), std::true_type(), std::true_type(), set_0); move_back(); }
        for (; kt + 1 < KT; advance()) { slice(stage, following(), std::false_type(), std::true_type(), set_0); move_back(); }
    }
    slice(stage, 0, std::false_type(), std::false_type(), set_0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// ---- epilogues: 8 columns from n on of row m; `some`: how many of them exist
// (what belongs to the columns is loaded once for all rows; bias: as it lies in memory)
struct column_pieces { u32x4 bias; float scale[8], scale_2[8]; };
struct column_terms { float bias[8], scale[8], scale_2[8]; };
__device__ __forceinline__ void load_column_pieces(const product_arguments &p, column_pieces &c, long n, int some) {
    if (p.bias) c.bias = load_guarded<2>((const char *)p.bias + 2 * n, 2 * some);
    if (p.b_scale) load_some<F32>(p.b_scale + n, some, c.scale);
    if (p.b2_scale) load_some<F32>(p.b2_scale + n, some, c.scale_2);
}
template <int Y>
__device__ __forceinline__ void widen_column_pieces(const product_arguments &p, const column_pieces &from, column_terms &c) {
    if (p.bias) widen<Y>(from.bias, c.bias);
#pragma unroll
    for (int i = 0; i < 8; i++) { c.scale[i] = from.scale[i]; c.scale_2[i] = from.scale_2[i]; }
}
// z: the product's sums; row_scale: of row m of a
__device__ __forceinline__ void scale_linear(const product_arguments &p, const column_terms &c, float (&z)[8], float row_scale) {
    if (p.a_scale) {
#pragma unroll
        for (int i = 0; i < 8; i++) z[i] *= row_scale * c.scale[i];
    }
    if (p.bias) {
#pragma unroll
        for (int i = 0; i < 8; i++) z[i] += c.bias[i];
    }
}
template <int Y>
__device__ __forceinline__ void load_residual(const product_arguments &p, float (&r)[8], long m, long n, int some) {
    load_some<Y>((const stored<Y> *)p.residual + m * p.ldr + n, some, r);
}
template <int Y>
__device__ __forceinline__ void store_linear(const product_arguments &p, const float (&z)[8], long m, long n, int some) {
    typedef stored<Y> T;
    if (m < p.rows_above) store_some<Y>((T *)p.y + m * p.N + n, some, z);
    else if (m >= p.split_row) store_some<Y>((T *)p.y_below + (m - p.split_row) * p.N + n, some, z);
}
template <int Y>
__device__ __forceinline__ void finish_linear(const product_arguments &p, const column_terms &c, float (&z)[8], const float (&r)[8], float row_scale, long m, long n,
                                              int some) {
    scale_linear(p, c, z, row_scale);
    if (p.pre) store_some<Y>((stored<Y> *)p.pre + m * p.N + n, some, z);
    activate(p.activation, z);
    if (p.residual) {
#pragma unroll
        for (int i = 0; i < 8; i++) z[i] += r[i];
    }
    store_linear<Y>(p, z, m, n, some);
}
template <int Y>
__device__ __forceinline__ void finish_gated(const product_arguments &p, const column_terms &c, float (&g)[8], float (&u)[8], float row_scale, long m, long n, int some) {
    typedef stored<Y> T;
    if (p.a_scale) {
#pragma unroll
        for (int i = 0; i < 8; i++) { g[i] *= row_scale * c.scale[i]; u[i] *= row_scale * c.scale_2[i]; }
    }
    if (p.pre) {
        store_some<Y>((T *)p.pre + m * p.N + n, some, g);
        store_some<Y>((T *)p.pre2 + m * p.N + n, some, u);
    }
    activate(p.activation, g);
#pragma unroll
    for (int i = 0; i < 8; i++) g[i] *= u[i];
    store_some<Y>((T *)p.y + m * p.N + n, some, g);
}

// Workgroup id -> tile.  Consecutive workgroups go to the eight XCDs in turn, each with an L2 of its own: every XCD gets a run of consecutive
// tiles, and runs go down BAND rows of tiles before they move a column on (bf16 8192^3 with 2, 4, 8, 16: 787, 748, 748, 770 us).
constexpr int XCDS = 8;
__device__ __forceinline__ void tile_of(int id, int rows, int columns, int &row, int &column) {
    const int tiles = rows * columns, each = tiles / XCDS, rest = tiles % XCDS, x = id % XCDS;
    id = x * each + (x < rest ? x : rest) + id / XCDS;
    constexpr int BAND = 4;
    const int band = id / (BAND * columns), in = id - band * BAND * columns;
    const int height = rows - band * BAND < BAND ? rows - band * BAND : BAND;
    column = in / height;
    row = band * BAND + in - column * height;
}

#ifdef __HIP_DEVICE_COMPILE__               // (the host's compilation needs no body, and rejects a second one of the same configuration)
// Tile `id` of the product, of part `split` of k.  Y: type of bias, residual and outputs.
template <class C, int Y>
__device__ __forceinline__ void compute_tile(const product_arguments &p, int id, int split, lds_char *lds) {
    int row, column;
    tile_of(id, (p.M + C::BM - 1) / C::BM, (p.N + C::COLUMNS - 1) / C::COLUMNS, row, column);
    const long m0 = (long)row * C::BM, n0 = (long)column * C::COLUMNS;
    constexpr int F = C::F, REGISTERS = F * F / 64;
    typename block_sums<F>::type acc[C::TM][C::TN];
#pragma unroll
    for (int i = 0; i < C::TM; i++)
#pragma unroll
        for (int j = 0; j < C::TN; j++)
#pragma unroll
            for (int r = 0; r < REGISTERS; r++) acc[i][j][r] = 0.f;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / C::WGN, wn = wave % C::WGN;
    constexpr int SPAN = C::EPILOGUE == GATED ? C::WN / 2 : C::WN;         // columns of C of a wavefront
    constexpr int ACROSS = SPAN / 8, DOWN = 64 / ACROSS;                   // lanes along a row, rows of one pass
    constexpr int PASSES = 32 / DOWN, STRIPS = C::WM / 32;
    const int r0 = lane / ACROSS, c0 = 8 * (lane % ACROSS);
    const long n = n0 + wn * SPAN + c0;
    const int some = (int)min(8L, p.N - n);
    // Bias and scales, where there are registers for them ahead of the product, which then covers their way from memory (e4m3, loaded behind the product /
    // ahead of it: 1024 x 4096 x 1024 9.8 / 8.6 us, 3000 x 700 x 2000 12.8 / 11.9, 1024 x 2048 x 1024 6.8 / 6.3).  A lane holds the scales of rows lane % 32 of the strips.
    constexpr bool TERMS = C::A_ROWS && C::B_ROWS, EARLY = C::TM * C::TN * REGISTERS <= 64;
    column_pieces pieces;
    float row_scales[STRIPS];
    auto load_terms = [&] {
        if (!TERMS || p.partial) return;
        if (some > 0) load_column_pieces(p, pieces, n, some);
        if constexpr (C::E == F8)
#pragma unroll
            for (int i = 0; i < STRIPS; i++) {
                const long m = m0 + wm * C::WM + i * 32 + lane % 32;
                row_scales[i] = p.a_scale[min(m, p.M - 1L)];
            }
    };
    if constexpr (EARLY) load_terms();
    const long k0 = p.partial ? (long)split * p.slices_per_split * C::BK : 0;
    const long K = p.partial ? min((long)p.slices_per_split * C::BK, p.K - k0) : p.K;
    accumulate<C>(acc, p.a, p.lda, p.b, p.ldb, p.b2, p.ldb2, p.M, p.N, m0, n0, k0, K, lds);
    if constexpr (C::EPILOGUE == LINEAR && C::A_ROWS && !C::B_ROWS)        // (only the gradient of a gated layer's input has two)
        if (p.a_more) accumulate<C>(acc, p.a_more, p.lda, p.b_more, p.ldb_more, nullptr, 0, p.M, p.N, m0, n0, k0, K, lds);

    if constexpr (!EARLY) load_terms();
    column_terms columns;
    if (TERMS && some > 0 && !p.partial) widen_column_pieces<Y>(p, pieces, columns);

    // A wavefront's strips of 32 rows, through LDS of its own: stored by columns of the accumulators, read by rows.
    const int at = lane % F, group = lane / F;
    __attribute__((address_space(3))) float *const strip = (__attribute__((address_space(3))) float *)lds + wave * 32 * C::STRIP;
    typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
    auto order_lanes = [] {                                               // what the lanes of a wavefront pass to each other
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
#pragma unroll
    for (int i = 0; i < STRIPS; i++) {
        const long first = m0 + wm * C::WM + i * 32 + r0;                 // the lane's row of pass 0
        const bool across = some > 0;
        auto take = [&](int pass, int c, float (&v)[8]) {
            const f32x4 a = *(lds_f32x4 *)(strip + (pass * DOWN + r0) * C::STRIP + c), b = *(lds_f32x4 *)(strip + (pass * DOWN + r0) * C::STRIP + c + 4);
#pragma unroll
            for (int e = 0; e < 4; e++) { v[e] = a[e]; v[4 + e] = b[e]; }
        };
        // the residual's pieces are on their way while the strip is turned, where nothing else is to be done
        constexpr bool RESIDUAL = C::EPILOGUE == LINEAR && C::A_ROWS && C::B_ROWS;
        float r[RESIDUAL ? PASSES : 1][8];
        if constexpr (RESIDUAL)
            if (p.residual && !p.partial && !(p.pre || p.activation != NONE)) {
#pragma unroll
                for (int pass = 0; pass < PASSES; pass++)
                    if (across && first + pass * DOWN < p.M) load_residual<Y>(p, r[pass], first + pass * DOWN, n, some);
            }
#pragma unroll
        for (int b = 0; b < 32 / F; b++)
#pragma unroll
            for (int j = 0; j < C::TN; j++)
#pragma unroll
                for (int g = 0; g < REGISTERS / 4; g++) {
                    const auto &v = acc[i * (32 / F) + b][j];
                    *(lds_f32x4 *)(strip + (b * F + at) * C::STRIP + j * F + 8 * g + 4 * group) = f32x4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
                }
        order_lanes();
        auto row_scale = [&](int pass) { return C::E == F8 ? __shfl(row_scales[i], pass * DOWN + r0) : 1.f; };       // (by all lanes)
        if (p.partial) {
#pragma unroll 1
            for (int pass = 0; pass < PASSES; pass++) {
                const long m = first + pass * DOWN;
                if (!across || m >= p.M) continue;
                constexpr long PARTS = C::EPILOGUE == GATED ? 2 : 1;
                float *out = p.partial + ((long)split * PARTS * p.M + m) * p.N + n;
#pragma unroll
                for (int part = 0; part < PARTS; part++) {
                    float z[8];
                    take(pass, part * SPAN + c0, z);
                    store_some<F32>(out + part * (long)p.M * p.N, some, z);
                }
            }
        } else if constexpr (C::EPILOGUE == GATED) {
#pragma unroll 1
            for (int pass = 0; pass < PASSES; pass++) {
                float z[8], u[8];
                take(pass, c0, z);
                take(pass, SPAN + c0, u);
                const float scale = row_scale(pass);
                if (across && first + pass * DOWN < p.M) finish_gated<Y>(p, columns, z, u, scale, first + pass * DOWN, n, some);
            }
        } else {
            bool plain = true;
            if constexpr (RESIDUAL) plain = !(p.pre || p.activation != NONE);
            if (plain) {
#pragma unroll
                for (int pass = 0; pass < PASSES; pass++) {
                    const float scale = row_scale(pass);
                    if (!across || first + pass * DOWN >= p.M) continue;
                    float z[8];
                    take(pass, c0, z);
                    if constexpr (RESIDUAL) {
                        scale_linear(p, columns, z, scale);
                        if (p.residual) {
#pragma unroll
                            for (int e = 0; e < 8; e++) z[e] += r[pass][e];
                        }
                    }
                    store_linear<Y>(p, z, first + pass * DOWN, n, some);
                }
            } else {
                // (many instructions: not unrolled)
#pragma unroll 1
                for (int pass = 0; pass < PASSES; pass++) {
                    const float scale = row_scale(pass);
                    if (!across || first + pass * DOWN >= p.M) continue;
                    float z[8], r[8];
                    if (p.residual) load_residual<Y>(p, r, first + pass * DOWN, n, some);
                    take(pass, c0, z);
                    finish_linear<Y>(p, columns, z, r, scale, first + pass * DOWN, n, some);
                }
            }
        }
        order_lanes();
    }
}
#endif

// grid: (tiles, splits of k)
template <class C, int Y>
__global__ __launch_bounds__(C::NT) void product_kernel(product_arguments p) {
#ifdef __HIP_DEVICE_COMPILE__
    extern __shared__ __attribute__((aligned(16))) char shared_bytes[];
    compute_tile<C, Y>(p, blockIdx.x, blockIdx.y, (lds_char *)shared_bytes);
#endif
}

// Two products in one launch (both gradients of a layer), the second's tiles behind the first's: compute units that the last round of
// the first leaves idle begin with the second, and where it leaves some, with the sums of the bias's gradient.  `start`: the second's first workgroup, a
// multiple of the XCDs; `end`: that of the sums.
template <class C, class D, int Y>
__global__ __launch_bounds__(C::NT) void product_pair_kernel(product_arguments p, product_arguments q, column_sums sums, int tiles, int start, int end) {
#ifdef __HIP_DEVICE_COMPILE__
    static_assert(C::NT == D::NT, "one workgroup's size");
    extern __shared__ __attribute__((aligned(16))) char shared_bytes[];
    const int id = blockIdx.x;
    if (id < tiles) compute_tile<C, Y>(p, id, 0, (lds_char *)shared_bytes);
    else if (id >= end) sum_parts<Y, C::NT>(sums, id - end, (float *)shared_bytes);
    else if (id >= start) compute_tile<D, Y>(q, id - start, 0, (lds_char *)shared_bytes);
#endif
}

// The partial sums of a product whose k was split, added in order, and the epilogue on them: 8 columns to a thread.
template <int Y, int EPILOGUE>
__global__ __launch_bounds__(256) void finish_kernel(product_arguments p, int splits) {
    const long across = (p.N + 7) / 8, id = (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= across * p.M) return;
    const long m = id / across, n = 8 * (id - m * across);
    const int some = (int)min(8L, p.N - n);
    constexpr long PARTS = EPILOGUE == GATED ? 2 : 1;
    float z[8], u[8];
#pragma unroll
    for (int i = 0; i < 8; i++) z[i] = u[i] = 0.f;
    for (int s = 0; s < splits; s++) {
        const float *part = p.partial + ((long)s * PARTS * p.M + m) * p.N + n;
        float v[8];
        load_some<F32>(part, some, v);
#pragma unroll
        for (int i = 0; i < 8; i++) z[i] += v[i];
        if constexpr (EPILOGUE == GATED) {
            load_some<F32>(part + (long)p.M * p.N, some, v);
#pragma unroll
            for (int i = 0; i < 8; i++) u[i] += v[i];
        }
    }
    column_pieces pieces;
    column_terms columns;
    load_column_pieces(p, pieces, n, some);
    widen_column_pieces<Y>(p, pieces, columns);
    const float scale = p.a_scale ? p.a_scale[m] : 1.f;
    if constexpr (EPILOGUE == GATED) finish_gated<Y>(p, columns, z, u, scale, m, n, some);
    else {
        if (p.residual) load_residual<Y>(p, u, m, n, some);
        finish_linear<Y>(p, columns, z, u, scale, m, n, some);
    }
}

}  // namespace tops
#endif
