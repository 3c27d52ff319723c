// The dense product's epilogue (linear.hip, linear256.hip, linear_few.hip): y = act(z + b) + r, and the derivative of act
// for its gradient. Everything in fp32; the store rounds once.
#pragma once
#include "common.hpp"

namespace sphip {

// Phi(x) = (1 + erf(x / sqrt 2)) / 2 from the complementary error function of Abramowitz & Stegun 7.1.26:
// erfc(u) = (a1 t + .. + a5 t^5) exp(-u^2), t = 1 / (1 + p u), u = |x| / sqrt 2, absolute error below 1.5e-7.
// One exponential, one reciprocal and 6 FMAs: the library's erff is three times as long, and act_value runs once
// per output behind a matrix product (67 M outputs of a 16384 x 4096 product: 30 us of VALU work against 80 with erff).
__device__ __forceinline__ float phi_tail(float x, float& e) {
    const float u = fabsf(x) * 0.70710678118654752f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, u, 1.f));
    e = __expf(-u * u);
    float p = fmaf(1.061405429f, t, -1.453152027f);
    p = fmaf(p, t, 1.421413741f);
    p = fmaf(p, t, -0.284496736f);
    p = fmaf(p, t, 0.254829592f);
    return 0.5f * p * t * e;                       // Phi(-|x|)
}

__device__ __forceinline__ float act_value(float z, int act) {
    if (act == SPHIP_ACT_RELU) return z > 0.f ? z : (z != z ? z : 0.f);
    if (act == SPHIP_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
    if (act == SPHIP_ACT_GELU) {
        // z Phi(z) = max(z, 0) - |z| Phi(-|z|), the tail as in phi_tail with its factors in the constants; from |z| = 30 on it
        // is zero in fp32 (and infinity times zero is avoided). A NaN stays one in max(z, 0).
        const float m = fminf(fabsf(z), 30.f), w = m * 0.84932180028801904f;
        const float t = __builtin_amdgcn_rcpf(fmaf(0.23164188588f, m, 1.f));
        float p = fmaf(0.5307027145f, t, -0.7265760135f);
        p = fmaf(p, t, 0.7107068705f);
        p = fmaf(p, t, -0.142248368f);
        p = fmaf(p, t, 0.127414796f);
        return fmaf(-m, p * t * __builtin_amdgcn_exp2f(-(w * w)), z < 0.f ? 0.f : z);
    }
    return z;
}

// four at once, the choice of activation outside
__device__ __forceinline__ void act_value4(float (&v)[4], int act) {
    if (act == SPHIP_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = act_value(v[j], SPHIP_ACT_RELU);
    } else if (act == SPHIP_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = act_value(v[j], SPHIP_ACT_GELU);
    } else if (act == SPHIP_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = act_value(v[j], SPHIP_ACT_SILU);
    }
}

__device__ __forceinline__ float act_slope(float z, int act) {
    if (act == SPHIP_ACT_RELU) return z > 0.f ? 1.f : (z != z ? z : 0.f);
    if (act == SPHIP_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
        return s * fmaf(z, 1.f - s, 1.f);
    }
    if (act == SPHIP_ACT_GELU) {
        float e;
        const float q = phi_tail(z, e);
        return fmaf(z * e, 0.39894228040143268f, z > 0.f ? 1.f - q : q);
    }
    return 1.f;
}

__device__ __forceinline__ float load_as_f32(const void* p, int dt, int64_t i) {
    return dt == SPHIP_BF16 ? bf16_to_f32(((const bf16_t*)p)[i]) : ((const float*)p)[i];
}

struct Epilogue {
    const void* bias = nullptr;       // (M) or null
    const void* res = nullptr;        // (N, M), row stride ldr, or null
    void* out = nullptr;              // (N, M), row stride ldo
    void* z = nullptr;                // (N, M), row stride ldz, or null: z + b before the activation, as values of z_dt
    uint8_t* z_scales = nullptr;      // or, with scales, as codes of that format (whole tiles only: finish_rows)
    int64_t ldr = 0, ldo = 0, ldz = 0;
    int bias_dt = 0, res_dt = 0, out_dt = 0, z_dt = 0;
    int act = 0;
};

// four consecutive elements at any element-aligned address (the hardware splits what is not 8- or 16-byte aligned; still
// one instruction where element accesses would be four)
typedef unsigned u2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned u4_any __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ void load4_as_f32(const void* p, int dt, int64_t i, float (&v)[4]) {
    if (dt == SPHIP_BF16) {
        const u2_any u = *(const u2_any*)((const bf16_t*)p + i);
        v[0] = __uint_as_float(u.x << 16), v[1] = __uint_as_float(u.x & 0xffff0000u);
        v[2] = __uint_as_float(u.y << 16), v[3] = __uint_as_float(u.y & 0xffff0000u);
    } else {
        const u4_any u = *(const u4_any*)((const float*)p + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(u[j]);
    }
}
__device__ __forceinline__ void store4_from_f32(void* p, int dt, int64_t i, const float (&v)[4]) {
    if (dt == SPHIP_BF16)
        *(u2_any*)((bf16_t*)p + i) = (u2_any){(unsigned)f32_to_bf16(v[0]) | ((unsigned)f32_to_bf16(v[1]) << 16),
                                              (unsigned)f32_to_bf16(v[2]) | ((unsigned)f32_to_bf16(v[3]) << 16)};
    else *(u4_any*)((float*)p + i) = (u4_any){__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
}
// the same past the caches: what no kernel reads soon
__device__ __forceinline__ void store4_stream(void* p, int dt, int64_t i, const float (&v)[4]) {
    if (dt == SPHIP_BF16)
        __builtin_nontemporal_store((u2_any){(unsigned)f32_to_bf16(v[0]) | ((unsigned)f32_to_bf16(v[1]) << 16),
                                             (unsigned)f32_to_bf16(v[2]) | ((unsigned)f32_to_bf16(v[3]) << 16)}, (u2_any*)((bf16_t*)p + i));
    else
        __builtin_nontemporal_store((u4_any){__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])},
                                    (u4_any*)((float*)p + i));
}
__device__ __forceinline__ void store_from_f32(void* p, int dt, int64_t i, float v) {
    if (dt == SPHIP_BF16) ((bf16_t*)p)[i] = f32_to_bf16(v);
    else ((float*)p)[i] = v;
}

// outputs (n, m .. m + 3) of the accumulated product v; columns past M are left alone
__device__ __forceinline__ void epilogue4(const Epilogue& e, int64_t n, int m, int M, float (&v)[4]) {
    if (m + 3 < M) {
        if (e.bias != nullptr) {
            float b[4];
            load4_as_f32(e.bias, e.bias_dt, m, b);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += b[j];
        }
        if (e.z != nullptr && e.z_scales == nullptr) store4_from_f32(e.z, e.z_dt, n * e.ldz + m, v);
        act_value4(v, e.act);
        if (e.res != nullptr) {
            float r[4];
            load4_as_f32(e.res, e.res_dt, n * e.ldr + m, r);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += r[j];
        }
        store4_from_f32(e.out, e.out_dt, n * e.ldo + m, v);
        return;
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) {
        if (m + j >= M) continue;
        float t = v[j];
        if (e.bias != nullptr) t += load_as_f32(e.bias, e.bias_dt, m + j);
        if (e.z != nullptr && e.z_scales == nullptr) store_from_f32(e.z, e.z_dt, n * e.ldz + m + j, t);
        t = act_value(t, e.act);
        if (e.res != nullptr) t += load_as_f32(e.res, e.res_dt, n * e.ldr + m + j);
        store_from_f32(e.out, e.out_dt, n * e.ldo + m + j, t);
    }
}

}  // namespace sphip
