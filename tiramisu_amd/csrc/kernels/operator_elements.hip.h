// Element types, activations and small pieces that the kernels of the transformer operators (rms_norm.hip.h, linear_tiles.hip.h,
// linear_few_tokens.hip.h) share.  Everything is computed in fp32; elements are widened when they are read and rounded once, to nearest
// even, when they are stored.
#ifndef TIRAMISU_AMD_OPERATOR_ELEMENTS_HIP_H
#define TIRAMISU_AMD_OPERATOR_ELEMENTS_HIP_H
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tops {

// Numbers of tiramisu_hip_wrappers.h
enum element : int { F32 = 0, F16 = 1, BF16 = 2, F8 = 3 };
enum activation : int { NONE = 0, RELU = 1, GELU = 2, GELU_TANH = 3, SILU = 4 };
constexpr float E4M3_MOST = 448.f;

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
// the same pieces at any address (rows of an odd number of elements)
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(1)));

template <int E> struct storage;
template <> struct storage<F32> { typedef float type; };
template <> struct storage<F16> { typedef _Float16 type; };
template <> struct storage<BF16> { typedef __bf16 type; };
template <> struct storage<F8> { typedef uint8_t type; };
template <int E> using stored = typename storage<E>::type;

// n elements (16 bytes of them, 8 of the 16-bit types where `n` is 8) at any address, as fp32 and back
template <int E, int N>
__device__ __forceinline__ void load_elements(const stored<E> *p, float (&v)[N]) {
    if constexpr (E == F32) {
        static_assert(N % 4 == 0, "whole 16-byte pieces");
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const u32x4 w = *reinterpret_cast<const u32x4_any *>(p + i);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const uint32_t word = w[c];              // (an element of a vector, given to the cast by itself, came out as another one)
                v[i + c] = __builtin_bit_cast(float, word);
            }
        }
    } else {
        static_assert(N % 8 == 0, "whole 16-byte pieces");
        typedef stored<E> pair __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            const u32x4 w = *reinterpret_cast<const u32x4_any *>(p + i);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const uint32_t word = w[c];
                const pair e = __builtin_bit_cast(pair, word);
                v[i + 2 * c] = (float)e[0];
                v[i + 2 * c + 1] = (float)e[1];
            }
        }
    }
}

template <int E, int N>
__device__ __forceinline__ void store_elements(stored<E> *p, const float (&v)[N]) {
    if constexpr (E == F32) {
#pragma unroll
        for (int i = 0; i < N; i += 4)
            *reinterpret_cast<u32x4_any *>(p + i) = u32x4{__builtin_bit_cast(uint32_t, v[i]), __builtin_bit_cast(uint32_t, v[i + 1]),
                                                          __builtin_bit_cast(uint32_t, v[i + 2]), __builtin_bit_cast(uint32_t, v[i + 3])};
    } else if constexpr (E == F8) {
        static_assert(N % 4 == 0, "whole words");
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[i], v[i + 1], 0, false);
            w = __builtin_amdgcn_cvt_pk_fp8_f32(v[i + 2], v[i + 3], w, true);
            typedef int int_any __attribute__((aligned(1)));
            *reinterpret_cast<int_any *>(p + i) = w;
        }
    } else {
        static_assert(N % 8 == 0, "whole 16-byte pieces");
        typedef stored<E> pair __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            u32x4 w;
#pragma unroll
            for (int c = 0; c < 4; c++) w[c] = __builtin_bit_cast(uint32_t, pair{(stored<E>)v[i + 2 * c], (stored<E>)v[i + 2 * c + 1]});
            *reinterpret_cast<u32x4_any *>(p + i) = w;
        }
    }
}

template <int E> __device__ __forceinline__ float load_one(const stored<E> *p) { return (float)*p; }
template <int E> __device__ __forceinline__ void store_one(stored<E> *p, float v) {
    if constexpr (E == F8) *p = (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xff);
    else *p = (stored<E>)v;
}

// The first `n` of N elements; the others count as zero and are not touched.
template <int E, int N>
__device__ __forceinline__ void load_some(const stored<E> *p, int n, float (&v)[N]) {
    if (n >= N) return load_elements<E>(p, v);
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = i < n ? load_one<E>(p + i) : 0.f;
}
template <int E, int N>
__device__ __forceinline__ void store_some(stored<E> *p, int n, const float (&v)[N]) {
    if (n >= N) return store_elements<E>(p, v);
#pragma unroll
    for (int i = 0; i < N; i++)
        if (i < n) store_one<E>(p + i, v[i]);
}

// 16 bytes at `p` of which `left` exist; the others are zero and not read
template <int BYTES>
__device__ __forceinline__ u32x4 load_guarded(const char *p, long left) {
    if (left >= 16) return *reinterpret_cast<const u32x4_any *>(p);
    u32x4 w = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16 / BYTES; i++)
        if (i * BYTES < left) {
            const uint32_t e = BYTES == 4 ? *reinterpret_cast<const uint32_t *>(p + 4 * i) : BYTES == 2 ? (uint32_t)*reinterpret_cast<const uint16_t *>(p + 2 * i)
                                                                                           : (uint32_t)*reinterpret_cast<const uint8_t *>(p + i);
            w[i * BYTES / 4] |= e << (8 * (i * BYTES % 4));
        }
    return w;
}

// ... as fp32
template <int E, int N>
__device__ __forceinline__ void widen(u32x4 w, float (&v)[N]) {
    static_assert(N == (E == F32 ? 4 : 8), "16 bytes");
#pragma unroll
    for (int c = 0; c < 4; c++) {
        const uint32_t word = w[c];                          // (an element of a vector, given to the cast by itself, came out as another one)
        if constexpr (E == F32) v[c] = __builtin_bit_cast(float, word);
        else {
            typedef stored<E> pair __attribute__((ext_vector_type(2)));
            const pair e = __builtin_bit_cast(pair, word);
            v[2 * c] = (float)e[0];
            v[2 * c + 1] = (float)e[1];
        }
    }
}

// ---- activations and their slopes.  exp2 of a large argument is infinite and 1 / infinity zero: silu and the sigmoid of the tanh form
// end at 0 and z without a comparison, and a NaN stays one.
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.442695041f * z)); }
__device__ __forceinline__ float gelu_tanh_argument(float z) { return 1.5957691216f * (z + 0.044715f * z * z * z); }   // 2 sqrt(2 / pi): 0.5 (1 + tanh a) = sigmoid(2 a)

// The normal distribution's lower tail at -|z|, 0.5 erfc(|z| / sqrt 2) = exp(-z^2 / 2) R(t) with t = 1 / (1 + 0.31 |z|), and exp(-z^2 / 2).  R is t times a
// polynomial of degree 5, fitted here to the smallest relative error (4.7e-6 up to |z| = 14, where the tail is below fp32's numbers; half a unit of
// float16 is 2.4e-4): relative, so that gelu of a large negative z, z times the tail, keeps its digits.  gelu(z) = max(z, 0) - |z| tail; the tail is zero
// from z = 16 on, and must not meet an infinite z there.
// (Epilogues are bound by these instructions: 3 million gelu cost 5 us with 17 of them and two of a quarter of the rate.)
__device__ __forceinline__ float normal_tail(float z, float &bell) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.31f, fabsf(z), 1.f));
    bell = __builtin_amdgcn_exp2f(-0.72134752044f * z * z);
    float r = -0.0739265304f;
    r = __builtin_fmaf(r, t, 0.180442905f);
    r = __builtin_fmaf(r, t, 0.0157528392f);
    r = __builtin_fmaf(r, t, 0.133425542f);
    r = __builtin_fmaf(r, t, 0.120442332f);
    r = __builtin_fmaf(r, t, 0.123860602f);
    return r * t * bell;
}

__device__ __forceinline__ float activated(int a, float z) {
    if (a == RELU) return z < 0.f ? 0.f : z;
    if (a == GELU) {
        float bell;
        return __builtin_fmaf(-fabsf(fminf(z, 16.f)), normal_tail(z, bell), fmaxf(z, 0.f));
    }
    return z * sigmoid(a == GELU_TANH ? gelu_tanh_argument(z) : z);
}
// (the choice is made once for all elements, whose instructions then cover each other)
template <int N>
__device__ __forceinline__ void activate(int a, float (&v)[N]) {
    if (a == GELU) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = activated(GELU, v[i]);
    } else if (a == SILU) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = activated(SILU, v[i]);
    } else if (a == GELU_TANH) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = activated(GELU_TANH, v[i]);
    } else if (a == RELU) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = activated(RELU, v[i]);
    }
}

// slope of the activation at z, and where `value` is asked for the activation itself
__device__ __forceinline__ float activation_slope(int a, float z, float &value) {
    if (a == RELU) { value = z < 0.f ? 0.f : z; return z > 0.f ? 1.f : z == z ? 0.f : z; }
    if (a == GELU) {
        float bell;
        const float tail = normal_tail(z, bell), p = z < 0.f ? tail : 1.f - tail;
        value = z * p;
        return p + z * 0.3989422804f * bell;
    }
    if (a == GELU_TANH) {
        const float s = sigmoid(gelu_tanh_argument(z));
        value = z * s;
        const float q = fminf(fabsf(z), 16.f);               // s (1 - s) is zero from there on, and must not meet an infinite square
        return s + z * s * (1.f - s) * 1.5957691216f * (1.f + 0.134145f * q * q);
    }
    if (a == SILU) {
        const float s = sigmoid(z);
        value = z * s;
        return s * (1.f + z * (1.f - s));
    }
    value = z;
    return 1.f;
}
template <int N>
__device__ __forceinline__ void activation_slopes(int a, const float (&z)[N], float (&slope)[N], float (&value)[N]) {
    auto all = [&](int known) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < N; i++) slope[i] = activation_slope(known, z[i], value[i]);
    };
    if (a == GELU) all(GELU);
    else if (a == SILU) all(SILU);
    else if (a == GELU_TANH) all(GELU_TANH);
    else if (a == RELU) all(RELU);
    else all(NONE);
}

// out[c] = sum over `parts` rows of partial[][c], in a fixed order: 32 columns to a workgroup, THREADS / 32 threads down each.  `s`: 33 floats for each of these.
struct column_sums {
    const float *partial;                   // [parts][columns]
    void *out;
    long columns;
    int parts;                              // 0: no sums
};
constexpr int SUM_COLUMNS = 32;
template <int E, int THREADS, typename FLOATS>
__device__ __forceinline__ void sum_parts(const column_sums &a, int id, FLOATS *s) {
    constexpr int DOWN = THREADS / SUM_COLUMNS;
    const int x = threadIdx.x % SUM_COLUMNS, y = threadIdx.x / SUM_COLUMNS;
    const long first = (long)id * SUM_COLUMNS, c = first + x;
    float v = 0.f;
    if (c < a.columns) {
#pragma unroll 8
        for (int p = y; p < a.parts; p += DOWN) v += a.partial[(long)p * a.columns + c];
    }
    s[y * (SUM_COLUMNS + 1) + x] = v;
    __syncthreads();
    const int column = threadIdx.x / DOWN, part = threadIdx.x % DOWN;
    v = s[part * (SUM_COLUMNS + 1) + column];
#pragma unroll
    for (int o = DOWN / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if (part == 0 && first + column < a.columns) store_one<E>((stored<E> *)a.out + first + column, v);
}

}  // namespace tops
#endif
