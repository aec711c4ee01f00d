// The 8-bit form of an activation kept between forward and backward (equss_ckpt_pack and its readers): 32 consecutive channels
// of a row share one scale byte b, which stands for 2^(b - 127); a code is an int8 or an e4m3 number.
// The scale is a power of two on purpose: dividing by it and multiplying with it round nothing in fp32, an int8 or e4m3 number
// times it is exact in bf16, and so the MFMA products of the backward pass read exactly the values that were kept.  What that
// costs against a scale that puts the largest magnitude on the format's end is one bit at most, and on average half of one;
// blocks of 32 give it back (a block's largest value bounds only its own 31 neighbours).
#pragma once
#include "equss_common.h"

namespace equss {

constexpr int kCkptBlock = 32;
constexpr int kCkptMinExp = -110;      // smallest scale exponent: what is kept, e4m3's subnormals included, is a normal fp32 / bf16
// Scale byte of a block that held an infinity or a NaN.  Its codes are 0, or, where signs are kept, a code of the value's sign:
// -1 or 1 in int8, a NaN of that sign in e4m3.  255 << 23 is an infinity, times code 0 a NaN; ckpt_value_scale makes it a NaN
// whatever the code.  The products (gemm_tn_ckpt.hip) do without that: a lost block is infinities or NaN there.
constexpr int kCkptNanByte = 255;

__device__ __forceinline__ float ckpt_scale(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }
__device__ __forceinline__ float ckpt_value_scale(uint32_t byte) {
    return __builtin_bit_cast(float, byte == (uint32_t)kCkptNanByte ? 0x7fc00000u : byte << 23);
}

// code number I (0..3) of a dword, before scaling
template <bool E4M3>
__device__ __forceinline__ f32x4 ckpt_decode4(uint32_t w) {
    if constexpr (E4M3) {
        typedef float f32x2_t __attribute__((ext_vector_type(2)));
        const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        return f32x4{lo.x, lo.y, hi.x, hi.y};
    } else {
        const int v = (int)w;
        return f32x4{(float)(int8_t)v, (float)(int8_t)(v >> 8), (float)(int8_t)(v >> 16), (float)(int8_t)(v >> 24)};
    }
}

}  // namespace equss
