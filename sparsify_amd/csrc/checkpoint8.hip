// 8-bit checkpoint of an activation x (N, D): what a backward pass keeps of it.
//
// Groups of 32 consecutive tokens of ONE feature share a scale 2^e, kept as the byte e + 127. The large values of a
// residual stream sit in a few features at nearly all tokens, so a group holds values of one size, and no feature spoils
// the resolution of another (a scale per token and 32 features would). The tokens are also what the weight gradient
// dW = dz^T x contracts over: every 32 terms of its sum share a scale.
//   e     the smallest with max|x| / 2^e <= 127 (int8) or 448 (e4m3), at least -126 or -117: the smallest code
//         is then a normal number, 2^-126, in bf16 as in fp32
//   int8  q = x / 2^e rounded to nearest even, |q| <= 127: off by at most 2^(e-1), i.e. 1/128 of the group's maximum
//   e4m3  x / 2^e rounded to the nearest 8-bit float of 4 exponent and 3 mantissa bits (OCP, no infinities): off by at
//         most 2^-4 of the value (2^(e-10) below 2^(e-6))
// A power of two makes the division exact (one rounding per value) and code times scale a bf16 number exactly.
// keep_sign: a value other than zero keeps its sign, the smallest code in place of zero (a ReLU's mask).
// A group with an infinity or a NaN in it has scale byte 255 and restores as NaN throughout.
// Codes (32 ceil(N/32), ldq) and scales (ceil(N/32), ldq), ldq a multiple of 16 >= D; padding rows and columns are zeros.
//
// Bound: HBM. One thread owns V columns of a group and holds its 32 rows in registers (32 independent loads in flight),
// so x is read once: maximum, scale, codes.
#include "codes8.hpp"

namespace sphip {

template <typename T, int V> struct Cols;                 // V columns of one row, raw bits
template <int V> struct Cols<bf16_t, V> {
    unsigned w[(V + 1) / 2];
    __device__ __forceinline__ void load(const bf16_t* p, int n) {
#pragma unroll
        for (int j = 0; j < (V + 1) / 2; ++j) w[j] = 0;
        if (n >= V) __builtin_memcpy(w, p, V * 2);
        else
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j < n) w[j >> 1] |= (unsigned)p[j] << ((j & 1) * 16);
    }
    __device__ __forceinline__ unsigned magnitude(int j) const { return (j & 1 ? w[j >> 1] & 0x7fff0000u : (w[j >> 1] << 16) & 0x7fff0000u); }
    __device__ __forceinline__ float value(int j) const { return __uint_as_float(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16); }
};
template <int V> struct Cols<float, V> {
    float w[V];
    __device__ __forceinline__ void load(const float* p, int n) {
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = 0.f;
        if (n >= V) __builtin_memcpy(w, p, V * 4);
        else
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j < n) w[j] = p[j];
    }
    __device__ __forceinline__ unsigned magnitude(int j) const { return __float_as_uint(w[j]) & 0x7fffffffu; }
    __device__ __forceinline__ float value(int j) const { return w[j]; }
};

// biased exponent byte of the group's scale from the bits of its largest magnitude
template <int FMT> __device__ __forceinline__ unsigned scale_byte(unsigned top) {
    if (top >= 0x7f800000u) return 255u;
    // top = f 2^E: f 2^6 <= 127 (f 2^8 <= 448) for mantissas up to 1.984375 (1.75), one step coarser above
    const unsigned most = FMT == SPHIP_INT8 ? 0x7e0000u : 0x600000u;
    const int e = (int)(top >> 23) - (FMT == SPHIP_INT8 ? 6 : 8) + ((top & 0x7fffffu) > most ? 1 : 0);
    return (unsigned)max(e, FMT == SPHIP_INT8 ? 1 : 10);
}

template <typename T, int V, int FMT, bool KEEP>
__global__ __launch_bounds__(256) void checkpoint8_save_kernel(const T* __restrict__ x, int64_t ldx, uint8_t* __restrict__ codes,
                                                               uint8_t* __restrict__ scales, int64_t ldq, int64_t N, int D) {
    const int per_row = (int)(ldq / V);
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t grp = i / per_row;
    if (grp * 32 >= N) return;
    const int c0 = (int)(i % per_row) * V;
    const T* p = x + grp * 32 * ldx + c0;
    Cols<T, V> v[32];
    const int rows = (int)min((int64_t)32, N - grp * 32);
#pragma unroll
    for (int t = 0; t < 32; ++t) v[t].load(p + (int64_t)t * ldx, t < rows ? D - c0 : 0);
    unsigned top[V];
#pragma unroll
    for (int j = 0; j < V; ++j) top[j] = 0;
#pragma unroll
    for (int t = 0; t < 32; ++t)
#pragma unroll
        for (int j = 0; j < V; ++j) top[j] = max(top[j], v[t].magnitude(j));
    float inv[V];
    bool bad[V];
    uint8_t sb[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const unsigned b = scale_byte<FMT>(top[j]);
        sb[j] = (uint8_t)b;
        bad[j] = b == 255u;
        inv[j] = __uint_as_float((bad[j] ? 127u : 254u - b) << 23);          // 2^-e, a normal number: 1 <= b <= 249
    }
    __builtin_memcpy(scales + grp * ldq + c0, sb, V);
    uint8_t* q = codes + grp * 32 * ldq + c0;
#pragma unroll
    for (int t = 0; t < 32; ++t) {
        uint8_t o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float a = v[t].value(j);
            unsigned c;
            if (FMT == SPHIP_INT8) {
                // one rounding, to nearest even, by adding 1.5 2^23: the low byte is the two's complement code
                c = __float_as_uint(fmaf(a, inv[j], 12582912.f)) & 0xffu;
                if (KEEP && c == 0u && a != 0.f) c = a < 0.f ? 0xffu : 1u;
            } else {
                const float s = a * inv[j];
                c = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(s, s, 0, false) & 0xffu;
                if (KEEP && (c & 0x7fu) == 0u && a != 0.f) c = a < 0.f ? 0x81u : 1u;
            }
            o[j] = (uint8_t)(bad[j] ? 0x7fu : c);                            // (not read: the scale is NaN)
        }
        __builtin_memcpy(q + (int64_t)t * ldq, o, V);
    }
}

template <typename T, int V, int FMT>
__global__ __launch_bounds__(256) void checkpoint8_restore_kernel(const uint8_t* __restrict__ codes,
                                                                  const uint8_t* __restrict__ scales, int64_t ldq,
                                                                  T* __restrict__ out, int64_t ldo, int64_t N, int D) {
    constexpr int ROWS = 8;                                                  // rows of one group per thread
    const int per_row = (int)(ldq / V);
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t blk = i / per_row;
    if (blk * ROWS >= N) return;
    const int c0 = (int)(i % per_row) * V, n = D - c0;
    if (n <= 0) return;
    uint8_t sb[V], q[ROWS][V];
    __builtin_memcpy(sb, scales + (blk * ROWS / 32) * ldq + c0, V);
#pragma unroll
    for (int t = 0; t < ROWS; ++t) __builtin_memcpy(q[t], codes + (blk * ROWS + t) * ldq + c0, V);
    float s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = scale_value(sb[j]);
#pragma unroll
    for (int t = 0; t < ROWS; ++t) {
        const int64_t row = blk * ROWS + t;
        if (row >= N) break;
        T o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float f = FMT == SPHIP_INT8 ? (float)(int8_t)q[t][j] : __builtin_amdgcn_cvt_f32_fp8((int)q[t][j], 0);
            Elem<T>::store(o, j, f * s[j]);                                  // exact
        }
        T* p = out + row * ldo + c0;
        if (n >= V) __builtin_memcpy(p, o, sizeof(o));
        else
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (j < n) p[j] = o[j];
    }
}

template <typename T, int V>
static void launch_save(const void* x, int64_t ldx, int fmt, int keep, uint8_t* codes, uint8_t* scales, int64_t ldq, int64_t N,
                        int64_t D, unsigned blocks, hipStream_t s) {
#define SPHIP_SAVE(F, KP)                                                                                            \
    hipLaunchKernelGGL((checkpoint8_save_kernel<T, V, F, KP>), dim3(blocks), dim3(256), 0, s, (const T*)x, ldx, codes, \
                       scales, ldq, N, (int)D)
    if (fmt == SPHIP_INT8) {
        if (keep) SPHIP_SAVE(SPHIP_INT8, true);
        else SPHIP_SAVE(SPHIP_INT8, false);
    } else {
        if (keep) SPHIP_SAVE(SPHIP_E4M3, true);
        else SPHIP_SAVE(SPHIP_E4M3, false);
    }
#undef SPHIP_SAVE
}

static int check_codes(const char* what, const void* codes, const void* scales, int64_t ldq, int fmt, int dtype, int64_t N,
                       int64_t D) {
    SPHIP_REQUIRE(valid_dtype(dtype), SPHIP_EINVAL, "%s: bad dtype %d", what, dtype);
    SPHIP_REQUIRE(fmt == SPHIP_INT8 || fmt == SPHIP_E4M3, SPHIP_EINVAL, "%s: bad format %d", what, fmt);
    SPHIP_REQUIRE(codes && scales, SPHIP_EINVAL, "%s: null pointer", what);
    SPHIP_REQUIRE(N > 0 && D > 0 && N < (1ll << 31) - 256 && D < (1ll << 31) - 256, SPHIP_EINVAL, "%s: bad shape N=%lld D=%lld",
                  what, (long long)N, (long long)D);
    SPHIP_REQUIRE(ldq >= D && ldq % 16 == 0 && ((uintptr_t)codes & 15) == 0 && ((uintptr_t)scales & 15) == 0, SPHIP_EINVAL,
                  "%s: codes and scales need 16-byte aligned rows of at least D", what);
    return SPHIP_OK;
}

}  // namespace sphip

extern "C" int sphip_checkpoint8_save(const void* x, int dtype, int64_t ldx, int fmt, int keep_sign, uint8_t* codes,
                                      uint8_t* scales, int64_t ldq, int64_t N, int64_t D, void* stream) {
    using namespace sphip;
    const int st = check_codes("checkpoint8_save", codes, scales, ldq, fmt, dtype, N, D);
    if (st != SPHIP_OK) return st;
    SPHIP_REQUIRE(x && ((uintptr_t)x & (dtype_size(dtype) - 1)) == 0, SPHIP_EINVAL, "checkpoint8_save: null or misaligned x");
    SPHIP_REQUIRE(ldx >= D, SPHIP_EINVAL, "checkpoint8_save: ldx is shorter than a row");
    hipStream_t s = (hipStream_t)stream;
    const int64_t groups = cdiv(N, 32);
    const int V = dtype == SPHIP_BF16 ? 4 : 2;
    const int64_t blocks = cdiv(groups * (ldq / V), 256);
    SPHIP_REQUIRE(blocks < (1ll << 31), SPHIP_EUNSUPPORTED, "checkpoint8_save: grid too large");
    if (dtype == SPHIP_BF16) launch_save<bf16_t, 4>(x, ldx, fmt, keep_sign, codes, scales, ldq, N, D, (unsigned)blocks, s);
    else launch_save<float, 2>(x, ldx, fmt, keep_sign, codes, scales, ldq, N, D, (unsigned)blocks, s);
    SPHIP_CHECK_LAUNCH("checkpoint8_save");
    return SPHIP_OK;
}

extern "C" int sphip_checkpoint8_restore(const uint8_t* codes, const uint8_t* scales, int64_t ldq, int fmt, void* out,
                                         int dtype, int64_t ldo, int64_t N, int64_t D, void* stream) {
    using namespace sphip;
    const int st = check_codes("checkpoint8_restore", codes, scales, ldq, fmt, dtype, N, D);
    if (st != SPHIP_OK) return st;
    SPHIP_REQUIRE(out && ((uintptr_t)out & (dtype_size(dtype) - 1)) == 0, SPHIP_EINVAL, "checkpoint8_restore: null or misaligned out");
    SPHIP_REQUIRE(ldo >= D, SPHIP_EINVAL, "checkpoint8_restore: ldo is shorter than a row");
    hipStream_t s = (hipStream_t)stream;
    const int V = dtype == SPHIP_BF16 ? 8 : 4;
    const int64_t blocks = cdiv(cdiv(N, 8) * (ldq / V), 256);
    SPHIP_REQUIRE(blocks < (1ll << 31), SPHIP_EUNSUPPORTED, "checkpoint8_restore: grid too large");
#define SPHIP_RESTORE(T, V, F)                                                                                              \
    hipLaunchKernelGGL((checkpoint8_restore_kernel<T, V, F>), dim3((unsigned)blocks), dim3(256), 0, s, codes, scales, ldq,   \
                       (T*)out, ldo, N, (int)D)
    if (dtype == SPHIP_BF16) {
        if (fmt == SPHIP_INT8) SPHIP_RESTORE(bf16_t, 8, SPHIP_INT8);
        else SPHIP_RESTORE(bf16_t, 8, SPHIP_E4M3);
    } else {
        if (fmt == SPHIP_INT8) SPHIP_RESTORE(float, 4, SPHIP_INT8);
        else SPHIP_RESTORE(float, 4, SPHIP_E4M3);
    }
#undef SPHIP_RESTORE
    SPHIP_CHECK_LAUNCH("checkpoint8_restore");
    return SPHIP_OK;
}
