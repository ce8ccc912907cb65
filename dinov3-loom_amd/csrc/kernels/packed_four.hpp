// 4-bit values with a scale per block of 32 (include/dinov3_packed.h), in registers.
#pragma once
#include "packed.hpp"

namespace dhx {

// The float whose exponent is scale byte b's (what the conversions take).
__device__ __forceinline__ float scale_of(uint32_t b) { return __builtin_bit_cast(float, b << 23); }

// Codes of two values; which byte of `to` they go into is a constant.
template <int BYTE>
__device__ __forceinline__ uint32_t two_codes(uint32_t to, half2_t v, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(to, v, scale, BYTE);
}
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
template <int BYTE>
__device__ __forceinline__ uint32_t two_codes(uint32_t to, bf16x2_t v, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(to, v, scale, BYTE);
}

struct FourBits {
    uint32_t codes, scale;
};

// The codes of a lane's 8 values and their block's scale byte; four lanes, 4n .. 4n+3,
// hold a block (all of them are active).
template <class T>
__device__ __forceinline__ FourBits four_bits(typename Num<T>::v8 v) {
    typedef T v2 __attribute__((ext_vector_type(2)));
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    // The largest magnitude of the block, as the bits of a T: those of magnitudes are in
    // order, and what is not finite lies above all others.
    const uint4_t w = __builtin_bit_cast(uint4_t, v);
    u16x2 top = {};
#pragma unroll
    for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[e] & 0x7fff7fffu));
    uint32_t m = max((uint32_t)top[0], (uint32_t)top[1]);
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xb1, 0xf, 0xf, false));  // quad_perm 1, 0, 3, 2
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4e, 0xf, 0xf, false));  // quad_perm 2, 3, 0, 1
    const float largest = (float)__builtin_bit_cast(T, (uint16_t)m);
    const int exponent = (int)(__builtin_bit_cast(uint32_t, largest) >> 23);
    const bool odd = exponent == 255;
    const uint32_t byte = odd ? 255 : (uint32_t)max(exponent - 2, 0);
    const float scale = scale_of(byte);
    uint32_t c = 0;
    c = two_codes<0>(c, v2{v[0], v[1]}, scale);
    c = two_codes<1>(c, v2{v[2], v[3]}, scale);
    c = two_codes<2>(c, v2{v[4], v[5]}, scale);
    c = two_codes<3>(c, v2{v[6], v[7]}, scale);
    return FourBits{odd ? 0 : c, byte};
}

}  // namespace dhx
