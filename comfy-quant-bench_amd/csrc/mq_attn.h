// Shared by the attention kernels over a paged cache: MFMA operand types, conversions and lane exchanges.
#pragma once

#include "mq_device.h"
#include "mq_internal.h"

namespace mq {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();

// 8 values of 16 bits as the products take them.
struct Frag {
    uint32_t w[4];
};

template <int DT>
__device__ __forceinline__ f32x4 mfma16(const Frag& a, const Frag& b, f32x4 c) {
    if constexpr (DT == kDtF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Largest / sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48, in each of them.
__device__ __forceinline__ float max4(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __builtin_fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __builtin_fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum4(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Low (EL = 0) or high (1) 16 bits of a and b side by side.
template <int EL>
__device__ __forceinline__ uint32_t pair16(uint32_t a, uint32_t b) {
    return __builtin_amdgcn_perm(b, a, EL ? 0x07060302u : 0x05040100u);
}

// Bytes 0 .. 3 of w, signed, to fp32.
__device__ __forceinline__ void i8x4(uint32_t w, float (&f)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = static_cast<float>(static_cast<int8_t>(w >> (8 * j)));
}

// Two fp32 values that a bf16 holds exactly (integers below 256), packed.
__device__ __forceinline__ uint32_t bf16_exact2(float a, float b) {
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}

// An fp16 pair as the sum of two bf16 pairs, hi + lo: exact, an fp16's 11 bits being 8 and 3 (a subnormal
// fp16 is a normal bf16).
__device__ __forceinline__ void split_f16(uint32_t w, uint32_t* hi, uint32_t* lo) {
    const float a = f16_bits_to_f32(static_cast<uint16_t>(w & 0xffffu)), b = f16_bits_to_f32(static_cast<uint16_t>(w >> 16));
    const uint32_t ha = __float_as_uint(a) & 0xffff0000u, hb = __float_as_uint(b) & 0xffff0000u;
    *hi = __builtin_amdgcn_perm(hb, ha, 0x07060302u);
    // an infinity or NaN is all in hi: their difference would be NaN for an infinity
    const float la = __builtin_isfinite(a) ? a - __uint_as_float(ha) : 0.0f;
    const float lb = __builtin_isfinite(b) ? b - __uint_as_float(hb) : 0.0f;
    *lo = bf16_exact2(la, lb);
}

}  // namespace
}  // namespace mq
