// The 8-bit checkpoint's codes (checkpoint8.hip) and their values.
#pragma once
#include "common.hpp"

namespace sphip {

constexpr int64_t MAX_GROUPS = 1ll << 23;          // workgroups in a launch of up to 512 threads each: fewer than 2^32 work-items

// The last piece of a row may hold fewer elements than 16 bytes do. Its load is moved back to end where the row ends (rows of
// at least 16 bytes; a load per element, each waited for, took as long as the rest: saving 5001 x 1111 in 8 bits 10.1 us
// against 8.2), and the `bytes` in front that belong to the piece before are dropped, zeros behind.
__device__ __forceinline__ void drop_front(unsigned (&w)[4], int bytes) {
    uint64_t lo = ((uint64_t)w[1] << 32) | w[0], hi = ((uint64_t)w[3] << 32) | w[2];
    const int s = 8 * bytes;
    if (s >= 64) lo = hi >> (s - 64), hi = 0;
    else if (s > 0) lo = (lo >> s) | (hi << (64 - s)), hi >>= s;
    w[0] = (unsigned)lo, w[1] = (unsigned)(lo >> 32), w[2] = (unsigned)hi, w[3] = (unsigned)(hi >> 32);
}
// n >= 1 elements from p of a row that has fewer than 16 bytes
template <typename T> __device__ __forceinline__ void load_short(const T* p, int n, unsigned (&w)[4]) {
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = 0;
#pragma unroll
    for (int j = 0; j < E - 1; ++j) {
        if (j >= n) continue;
        if constexpr (sizeof(T) == 2) w[j / 2] |= (unsigned)p[j] << ((j & 1) * 16);
        else w[j] = __float_as_uint(p[j]);
    }
}

// 2^(byte - 127); byte 255 marks a group that held an infinity or a NaN: every value of it is NaN
__device__ __forceinline__ float scale_value(unsigned byte) {
    return __uint_as_float(byte == 255u ? 0x7fc00000u : byte << 23);
}

// The four codes of w, each under its own scale. int8: (u - 128) s with u the byte of w ^ 0x80808080 (128 s may be past the
// largest fp32: not u s - 128 s). Code times scale is exact in either format.
template <int FMT> __device__ __forceinline__ void code_values(unsigned w, const float (&s)[4], float (&o)[4]) {
    if (FMT == SPHIP_INT8) {
        w ^= 0x80808080u;
        o[0] = ((float)(w & 0xffu) - 128.f) * s[0];
        o[1] = ((float)((w >> 8) & 0xffu) - 128.f) * s[1];
        o[2] = ((float)((w >> 16) & 0xffu) - 128.f) * s[2];
        o[3] = ((float)(w >> 24) - 128.f) * s[3];
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

// The other direction. Biased exponent byte of a group's scale from the bits of its largest magnitude (255: a NaN or an
// infinity in it): the smallest that keeps top = f 2^E within the largest code, f 2^6 <= 127 (f 2^8 <= 448) up to a mantissa
// of 1.984375 (1.75), one step coarser above.
template <int FMT> __device__ __forceinline__ unsigned scale_byte(unsigned top) {
    if (top >= 0x7f800000u) return 255u;
    const unsigned most = FMT == SPHIP_INT8 ? 0x7e0000u : 0x600000u;
    const int e = (int)(top >> 23) - (FMT == SPHIP_INT8 ? 6 : 8) + ((top & 0x7fffffu) > most ? 1 : 0);
    return (unsigned)max(e, FMT == SPHIP_INT8 ? 1 : 10);
}
// 1 / scale, a normal number (1 <= byte <= 249)
__device__ __forceinline__ float inverse_scale(unsigned byte) { return __uint_as_float((byte == 255u ? 127u : 254u - byte) << 23); }
// Codes of four values, given the inverse scales: powers of two, so that a * inv is exact and there is one rounding, to
// nearest even. bad: 0xff in the bytes whose group is to read as NaN (their codes are not looked at; kept finite).
// Under the largest scale the next code up, 64 2^122 (256 2^120), is past the largest fp32: what would round to it, from
// 63.5 2^122 (248 2^120) on, is taken as the number just below, so that a finite value restores as one.
template <int FMT> __device__ __forceinline__ unsigned codes_of(const float (&v)[4], const float (&inv)[4], bool keep_sign, unsigned bad) {
    const float most = __uint_as_float(FMT == SPHIP_INT8 ? 0x7f7dffffu : 0x7f77ffffu);
    unsigned w;
    float a[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = __builtin_amdgcn_fmed3f(v[j], -most, most);
    if (FMT == SPHIP_INT8) {
        // + 1.5 2^23: the low byte is the two's complement code
        unsigned c[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = __float_as_uint(fmaf(a[j], inv[j], 12582912.f));
        const unsigned lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(c[3], c[2], 0x04000c0cu);
        w = lo | hi;
    } else {
        int t = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * inv[0], a[1] * inv[1], 0, false);
        w = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(a[2] * inv[2], a[3] * inv[3], t, true);
    }
    if (keep_sign) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned c = (w >> (8 * j)) & (FMT == SPHIP_INT8 ? 0xffu : 0x7fu);
            const unsigned least = FMT == SPHIP_INT8 ? (a[j] < 0.f ? 0xffu : 1u) : (a[j] < 0.f ? 0x81u : 1u);
            if (c == 0u && a[j] != 0.f) w = (w & ~(0xffu << (8 * j))) | (least << (8 * j));
        }
    }
    return (w & ~bad) | (bad & 0x7f7f7f7fu);
}

// Codes to values: a thread takes 16 bytes of values of 8 consecutive rows of one group (their loads all in flight).
struct RestoreArgs {
    const uint8_t *codes, *scales;
    void* out;
    int64_t ldq, ldo, N;
    int D;
};
static inline int64_t restore_blocks(const RestoreArgs& a, int dtype) { return cdiv(cdiv(a.N, 8) * (a.ldq / (16 / (int64_t)dtype_size(dtype))), 256); }
template <typename T, int FMT> __device__ __forceinline__ void restore_block(const RestoreArgs& a, unsigned block) {
    constexpr int ROWS = 8, V = 16 / sizeof(T);
    const int per_row = (int)(a.ldq / V);
    const int64_t i = (int64_t)block * 256 + threadIdx.x;
    const int64_t blk = i / per_row;
    if (blk * ROWS >= a.N) return;
    const int c0 = (int)(i % per_row) * V, n = a.D - c0;
    if (n <= 0) return;
    uint8_t sb[V], q[ROWS][V];
    __builtin_memcpy(sb, a.scales + (blk * ROWS / 32) * a.ldq + c0, V);
#pragma unroll
    for (int t = 0; t < ROWS; ++t) __builtin_memcpy(q[t], a.codes + (blk * ROWS + t) * a.ldq + c0, V);
    float s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = scale_value(sb[j]);
#pragma unroll
    for (int t = 0; t < ROWS; ++t) {
        const int64_t row = blk * ROWS + t;
        if (row >= a.N) break;
        T o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float f = FMT == SPHIP_INT8 ? (float)(int8_t)q[t][j] : __builtin_amdgcn_cvt_f32_fp8((int)q[t][j], 0);
            Elem<T>::store(o, j, f * s[j]);                                  // exact
        }
        T* p = (T*)a.out + row * a.ldo + c0;
        // past the caches (65536 x 4096 bf16 190 -> 125 us, 4096 x 4096 13.3 -> 7.3)
        typedef unsigned u4_out __attribute__((ext_vector_type(4), aligned(2)));
        if (n >= V) __builtin_nontemporal_store(__builtin_bit_cast(u4_out, o), (u4_out*)p);
        else
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j < n) p[j] = o[j];
    }
}

}  // namespace sphip
