// e4m3: 8-bit floats with 3 bits of fraction, 2^-9 .. 448, no infinities, 0x7F and 0xFF NaN.
#pragma once

#include "dev_common.h"

namespace navi_amd {

struct f8_t {
    uint8_t b;
};

// Four values as four bytes, rounded to nearest (ties to even). Past 448, infinities too: 448 of its sign; NaN stays NaN.
__device__ __forceinline__ uint32_t f8_pack4(f32x4_t v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = fabsf(v[i]) > 448.f ? copysignf(448.f, v[i]) : v[i];
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true));
}

// Four bytes as four values of f16 or bf16, both of which hold every one exactly.
template <class E>
__device__ __forceinline__ void f8_unpack4(uint32_t w, uint32_t (&out)[2]);
template <>
__device__ __forceinline__ void f8_unpack4<_Float16>(uint32_t w, uint32_t (&out)[2]) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true);
    __builtin_memcpy(&out[0], &a, 4);
    __builtin_memcpy(&out[1], &b, 4);
}
template <>
__device__ __forceinline__ void f8_unpack4<__bf16>(uint32_t w, uint32_t (&out)[2]) {
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true);
    __builtin_memcpy(&out[0], &a, 4);
    __builtin_memcpy(&out[1], &b, 4);
}

// Whether one of 16 of them is NaN.
__device__ __forceinline__ bool f8_any_nan(u32x4_t x) {
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) b |= (x[i] & 0x7F7F7F7Fu) + 0x01010101u;
    return (b & 0x80808080u) != 0;
}

} // namespace navi_amd
