// The two 16-bit activation types of the decoder-attention operators as bit patterns: conversions
// and matrix products. FORGE_FP16 is the type of the INT8 path; FORGE_BF16 has the same products at
// the same rate.
#pragma once

#include "common.h"

namespace forge_amd {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

struct Fp16 {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    static constexpr uint32_t kOnes = 0x3C003C00u;
    static constexpr uint32_t kInfinity = 0x7C00u;
    static constexpr float kNormal = 0x1p-14f;   // the smallest number of all its bits
    static constexpr bool kWide = false;   // FP32's range
    static __device__ __forceinline__ float widen(uint16_t b) { return h2f(b); }
    // Two values rounded to nearest even, the first in the low half. (No inline asm: the wait state between an
    // exponential and its use is the compiler's to keep.)
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{a, b}), v2));
    }
    // c + both values of the pair
    static __device__ __forceinline__ float add_pair(uint32_t p, float c) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, p), __builtin_bit_cast(v2, kOnes), c, false);
    }
    // c, or NaN if one of the pair is no finite number
    static __device__ __forceinline__ float times_zero(uint32_t p, float c) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, p), __builtin_bit_cast(v2, 0u), c, false);
    }
    static __device__ __forceinline__ v4f mfma16(v4u a, v4u b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ v16f mfma32(v4u a, v4u b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
};

struct Bf16 {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    static constexpr uint32_t kOnes = 0x3F803F80u;
    static constexpr uint32_t kInfinity = 0x7F80u;
    static constexpr float kNormal = 0x1p-126f;
    static constexpr bool kWide = true;
    static __device__ __forceinline__ float widen(uint16_t b) { return __uint_as_float(static_cast<uint32_t>(b) << 16); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f{a, b}), v2));
    }
    static __device__ __forceinline__ float add_pair(uint32_t p, float c) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, p), __builtin_bit_cast(v2, kOnes), c, false);
    }
    static __device__ __forceinline__ float times_zero(uint32_t p, float c) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, p), __builtin_bit_cast(v2, 0u), c, false);
    }
    static __device__ __forceinline__ v4f mfma16(v4u a, v4u b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ v16f mfma32(v4u a, v4u b, v16f c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
    }
};

template <class T>
__device__ __forceinline__ uint16_t narrow(float f) {
    return static_cast<uint16_t>(T::pack(f, f) & 0xFFFFu);
}
template <class T>
__device__ __forceinline__ void widen8(v4u v, float (&f)[8]) {
#pragma unroll
    for (int d = 0; d < 4; d++) {
        f[2 * d] = T::widen(static_cast<uint16_t>(v[d] & 0xFFFFu));
        f[2 * d + 1] = T::widen(static_cast<uint16_t>(v[d] >> 16));
    }
}
template <class T>
__device__ __forceinline__ v4u narrow8(const float (&f)[8]) {
    return v4u{T::pack(f[0], f[1]), T::pack(f[2], f[3]), T::pack(f[4], f[5]), T::pack(f[6], f[7])};
}

}  // namespace forge_amd
