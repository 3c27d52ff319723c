// Values of the 8-bit checkpoint codes (checkpoint8.hip).
#pragma once
#include "common.hpp"

namespace sphip {

// 2^(byte - 127); byte 255 marks a group that held an infinity or a NaN: every value of it is NaN
__device__ __forceinline__ float scale_value(unsigned byte) {
    return __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23);
}

// The four codes of w, each under its own scale. int8: (u - 128) s with u the byte of w ^ 0x80808080, as one fused
// u s - 128 s. Code times scale is exact in either format.
template <int FMT> __device__ __forceinline__ void code_values(unsigned w, const float (&s)[4], float (&o)[4]) {
    if (FMT == SPHIP_INT8) {
        w ^= 0x80808080u;
        o[0] = fmaf((float)(w & 0xffu), s[0], -128.f * s[0]);
        o[1] = fmaf((float)((w >> 8) & 0xffu), s[1], -128.f * s[1]);
        o[2] = fmaf((float)((w >> 16) & 0xffu), s[2], -128.f * s[2]);
        o[3] = fmaf((float)(w >> 24), s[3], -128.f * s[3]);
    } else {
        typedef float f2 __attribute__((ext_vector_type(2)));
        const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        o[0] = a.x * s[0], o[1] = a.y * s[1], o[2] = b.x * s[2], o[3] = b.y * s[3];
    }
}
template <int FMT> __device__ __forceinline__ void code_values(unsigned w, float s, float (&o)[4]) {
    const float s4[4] = {s, s, s, s};
    code_values<FMT>(w, s4, o);
}

}  // namespace sphip
