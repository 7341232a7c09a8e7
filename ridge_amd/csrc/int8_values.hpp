// int8_values.hpp -- values of rows in registers: loads and stores of several elements at once,
// and the rounding of a row to 8 bits.
#pragma once

#include <hip/hip_runtime.h>

#include <cfloat>
#include <cstdint>

namespace ridge {

// n elements of a row at once, with the alignment of one: rows may start anywhere, and
// global accesses of any alignment are one instruction here. What a row has behind its
// last whole vector goes one element a lane.
template <typename T, int n>
struct Memory {
    typedef T Vec __attribute__((ext_vector_type(n), aligned(sizeof(T))));
};

// STREAM: past the caches. A template argument, because the compiler merges the two
// accesses of a run-time choice and drops the hint.
template <bool STREAM, int n, typename T>
__device__ __forceinline__ void loadRow(const T* at, float (&v)[n]) {
    typedef typename Memory<T, n>::Vec Vec;
    Vec m;
    if constexpr (STREAM && n > 1) {
        m = __builtin_nontemporal_load((const Vec*)at);
    } else {
        m = *(const Vec*)at;
    }
#pragma unroll
    for (int e = 0; e < n; ++e) v[e] = (float)m[e];
}

template <bool STREAM, int n, typename T>
__device__ __forceinline__ void storeRow(T* at, const float (&v)[n]) {
    typedef typename Memory<T, n>::Vec Vec;
    Vec m;
#pragma unroll
    for (int e = 0; e < n; ++e) m[e] = (T)v[e];
    if constexpr (STREAM && n > 1) {
        __builtin_nontemporal_store(m, (Vec*)at);
    } else {
        *(Vec*)at = m;
    }
}

// A row's 127th: the largest magnitude over 127 is whole + rest to about 46 bits.
struct Step {
    float whole, rest, inverse;   // and 1 / whole
};

// Nearest whole numbers (halves to even) of v / step. The quotient is v * (1 / step) corrected
// once by its remainder, which is exact but for what `rest` lacks, so that a quotient of n + 1/2
// comes out as that: by the step's f32 alone, half of a row's largest value (63.5) went to 63
// or to 64 as the step was rounded. Adding 1.5 * 2^23 leaves the whole number in the low bits.
// A row whose scale is not finite gets bytes that mean nothing.
template <int n>
__device__ __forceinline__ void storeRounded(int8_t* at, const float (&v)[n], const Step& step) {
    typename Memory<signed char, n>::Vec b;
#pragma unroll
    for (int e = 0; e < n; ++e) {
        float t = v[e] * step.inverse;
        t = fmaf(fmaf(-t, step.rest, fmaf(-t, step.whole, v[e])), step.inverse, t);
        b[e] = (signed char)__float_as_uint(t + 12582912.0f);
    }
    *(typename Memory<signed char, n>::Vec*)at = b;
}

// Magnitudes are compared as integers: that is their order, and a NaN is above all.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

constexpr float kLift = 0x1p64f, kSmallRow = 0x1p-60f;

// The scale of a row whose largest magnitude is `most` before `root` multiplies it, and the step
// of its values before that: q is value / (most / 127), where the root is in both and cancels.
// Rows of small values are lifted by a power of two, so that the step's rest stays a normal
// number: the values of a row with most < kSmallRow go in times kLift.
__device__ __forceinline__ Step stepOf(float most, float root, float& scale) {
    scale = most * root / 127.0f;
    const bool small = most < kSmallRow;
    const float lifted = small ? most * kLift : most;
    Step step;
    step.whole = lifted / 127.0f;
    step.rest = fmaf(-127.0f, step.whole, lifted) / 127.0f;
    if (scale < FLT_MIN) {  // a NaN stays one
        scale = FLT_MIN;
        step.whole = (small ? FLT_MIN * kLift : FLT_MIN) / root;
        step.rest = 0.0f;
    }
    step.inverse = 1.0f / step.whole;
    return step;
}

}  // namespace ridge
