// 8-bit checkpoint of an activation x (N, D): what a backward pass keeps of it.
//
// Groups of 32 consecutive tokens of ONE feature share a scale 2^e, kept as the byte e + 127. The large values of a
// residual stream sit in a few features at nearly all tokens, so a group holds values of one size, and no feature spoils
// the resolution of another (a scale per token and 32 features would). The tokens are also what the weight gradient
// dW = dz^T x contracts over: every 32 terms of its sum share a scale.
//   e     the smallest with max|x| / 2^e <= 127 (int8) or 448 (e4m3), at least -126 or -117: the smallest code
//         is then a normal number, 2^-126, in bf16 as in fp32
//   int8  q = x / 2^e rounded to nearest even, |q| <= 127: off by at most 2^(e-1), above the smallest scale at most 1/127 of
//         the group's maximum (which is more than 63.5 steps)
//   e4m3  x / 2^e rounded to the nearest 8-bit float of 4 exponent and 3 mantissa bits (OCP, no infinities): off by at
//         most 2^-4 of the value (2^(e-10) below 2^(e-6))
// Values from 63.5 2^122 (248 2^120) on, whose nearest code would stand for 2^128, take the code below: finite (codes_of).
// A power of two makes the division exact (one rounding per value) and code times scale a bf16 number exactly.
// keep_sign: a value other than zero keeps its sign, the smallest code in place of zero (a ReLU's mask).
// A group with an infinity or a NaN in it has scale byte 255 and restores as NaN throughout.
// Codes (32 ceil(N/32), ldq) and scales (ceil(N/32), ldq), ldq a multiple of 16 >= D; padding rows and columns are zeros.
//
// Bound: HBM. A workgroup takes a group's 32 rows of 32 x 16 bytes of columns: 32 lanes side by side, every thread 4 rows,
// all loads in flight at once; x is read once, its maxima meet in LDS. (A thread per column piece and all 32 rows, no LDS,
// has an eighth of the threads: as fast at 65536 x 4096, 20 us against 8 at 5001 x 1111.)
#include "codes8.hpp"

namespace sphip {

struct SaveArgs {
    const void* x;
    uint8_t *codes, *scales;
    void* packed;                  // or null: also a copy of x, rows of ldp (a multiple of 64), zeros behind column D
    int64_t ldx, ldq, ldp, N;
    int D, strips, keep;           // strips: workgroups side by side along a row
};

template <typename T, int FMT>
__global__ __launch_bounds__(256) void checkpoint8_save_kernel(SaveArgs a) {
    constexpr int V = 16 / sizeof(T), W = 4;
    __shared__ unsigned red[4][32 * V];
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5, wave = threadIdx.x >> 6;
    const int64_t grp = blockIdx.x / (unsigned)a.strips, r0 = grp * 32 + rl;
    const int c0 = ((int)(blockIdx.x % (unsigned)a.strips) * 32 + cl) * V, n = a.D - c0;
    const int miss = max(V - n, 0);                              // (see drop_front)
    unsigned w[W][4];                                            // 4 rows of 16 bytes, raw
#pragma unroll
    for (int t = 0; t < W; ++t) {
        const int64_t row = r0 + 8 * t;
        const T* p = (const T*)a.x + row * a.ldx + c0;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[t][j] = 0;
        if (row >= a.N || n <= 0) continue;
        if (a.D >= V) __builtin_memcpy(w[t], p - miss, 16);
        else load_short(p, n, w[t]);
    }
    if (miss > 0 && a.D >= V)
#pragma unroll
        for (int t = 0; t < W; ++t) drop_front(w[t], miss < V ? miss * (int)sizeof(T) : 0);
    // element j of a row as fp32 bits
    auto bits = [&](int t, int j) {
        if (sizeof(T) == 4) return w[t][j % 4];
        return j & 1 ? w[t][j / 2] & 0xffff0000u : w[t][j / 2] << 16;
    };
    unsigned top[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        top[j] = 0;
#pragma unroll
        for (int t = 0; t < W; ++t) top[j] = max(top[j], bits(t, j) & 0x7fffffffu);
        top[j] = max(top[j], (unsigned)__shfl_xor((int)top[j], 32, 64));
    }
    if ((rl & 1) == 0)
#pragma unroll
        for (int j = 0; j < V; j += 4) *reinterpret_cast<uint4*>(&red[wave][cl * V + j]) = make_uint4(top[j], top[j + 1], top[j + 2], top[j + 3]);
    __syncthreads();
    if (c0 >= max(a.ldq, a.packed != nullptr ? a.ldp : 0)) return;
    float inv[V / 4][4];
    unsigned bad[V / 4], sb[V / 4];
#pragma unroll
    for (int j = 0; j < V; j += 4) {
        bad[j / 4] = sb[j / 4] = 0;
        uint4 m = *reinterpret_cast<const uint4*>(&red[0][cl * V + j]);
#pragma unroll
        for (int i = 1; i < 4; ++i) {
            const uint4 o = *reinterpret_cast<const uint4*>(&red[i][cl * V + j]);
            m = make_uint4(max(m.x, o.x), max(m.y, o.y), max(m.z, o.z), max(m.w, o.w));
        }
        const unsigned mv[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned b = scale_byte<FMT>(mv[i]);
            sb[j / 4] |= b << (8 * i), bad[j / 4] |= b == 255u ? 0xffu << (8 * i) : 0u, inv[j / 4][i] = inverse_scale(b);
        }
    }
    const bool in = c0 < a.ldq;
    if (rl == 0 && in) __builtin_memcpy(a.scales + grp * a.ldq + c0, sb, V);
#pragma unroll
    for (int t = 0; t < W; ++t) {
        const int64_t row = r0 + 8 * t;
        if (in) {
            unsigned o[V / 4];
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                const float v[4] = {__uint_as_float(bits(t, j)), __uint_as_float(bits(t, j + 1)), __uint_as_float(bits(t, j + 2)),
                                    __uint_as_float(bits(t, j + 3))};
                o[j / 4] = codes_of<FMT>(v, inv[j / 4], a.keep != 0, bad[j / 4]);
            }
            // past the caches: they are for the backward pass (65536 x 4096 bf16 150 -> 143 us, 4096 x 4096 11.4 -> 8.6)
            if constexpr (V == 8) __builtin_nontemporal_store(((uint64_t)o[V / 8] << 32) | o[0], (uint64_t*)(a.codes + row * a.ldq + c0));
            else __builtin_nontemporal_store(o[0], (unsigned*)(a.codes + row * a.ldq + c0));
        }
        if (a.packed != nullptr && row < a.N && c0 < a.ldp)
            *reinterpret_cast<uint4*>((T*)a.packed + row * a.ldp + c0) = make_uint4(w[t][0], w[t][1], w[t][2], w[t][3]);
    }
}

template <typename T, int FMT> __global__ __launch_bounds__(256) void checkpoint8_restore_kernel(RestoreArgs a) {
    restore_block<T, FMT>(a, blockIdx.x);
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

// see linear.hpp
int save_codes(const char* what, const void* x, int dtype, int64_t ldx, int fmt, int keep_sign, uint8_t* codes, uint8_t* scales,
               int64_t ldq, void* packed, int64_t ldp, int64_t N, int64_t D, hipStream_t s) {
    const int V = dtype == SPHIP_BF16 ? 8 : 4;
    const int64_t strips = cdiv(packed && ldp > ldq ? ldp : ldq, 32 * V), blocks = cdiv(N, 32) * strips;
    SPHIP_REQUIRE(blocks < MAX_GROUPS, SPHIP_EUNSUPPORTED, "%s: grid too large", what);
    const SaveArgs a = {x, codes, scales, packed, ldx, ldq, ldp, N, (int)D, (int)strips, keep_sign};
    const dim3 grid((unsigned)blocks), block(256);
    if (dtype == SPHIP_BF16) {
        if (fmt == SPHIP_INT8) hipLaunchKernelGGL((checkpoint8_save_kernel<bf16_t, SPHIP_INT8>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((checkpoint8_save_kernel<bf16_t, SPHIP_E4M3>), grid, block, 0, s, a);
    } else {
        if (fmt == SPHIP_INT8) hipLaunchKernelGGL((checkpoint8_save_kernel<float, SPHIP_INT8>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((checkpoint8_save_kernel<float, SPHIP_E4M3>), grid, block, 0, s, a);
    }
    SPHIP_CHECK_LAUNCH(what);
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
    return save_codes("checkpoint8_save", x, dtype, ldx, fmt, keep_sign, codes, scales, ldq, nullptr, 0, N, D, (hipStream_t)stream);
}

extern "C" int sphip_checkpoint8_restore(const uint8_t* codes, const uint8_t* scales, int64_t ldq, int fmt, void* out,
                                         int dtype, int64_t ldo, int64_t N, int64_t D, void* stream) {
    using namespace sphip;
    const int st = check_codes("checkpoint8_restore", codes, scales, ldq, fmt, dtype, N, D);
    if (st != SPHIP_OK) return st;
    SPHIP_REQUIRE(out && ((uintptr_t)out & (dtype_size(dtype) - 1)) == 0, SPHIP_EINVAL, "checkpoint8_restore: null or misaligned out");
    SPHIP_REQUIRE(ldo >= D, SPHIP_EINVAL, "checkpoint8_restore: ldo is shorter than a row");
    hipStream_t s = (hipStream_t)stream;
    const RestoreArgs a = {codes, scales, out, ldq, ldo, N, (int)D};
    const int64_t blocks = restore_blocks(a, dtype);
    SPHIP_REQUIRE(blocks < MAX_GROUPS, SPHIP_EUNSUPPORTED, "checkpoint8_restore: grid too large");
#define SPHIP_RESTORE(T, F) hipLaunchKernelGGL((checkpoint8_restore_kernel<T, F>), dim3((unsigned)blocks), dim3(256), 0, s, a)
    if (dtype == SPHIP_BF16) {
        if (fmt == SPHIP_INT8) SPHIP_RESTORE(bf16_t, SPHIP_INT8);
        else SPHIP_RESTORE(bf16_t, SPHIP_E4M3);
    } else {
        if (fmt == SPHIP_INT8) SPHIP_RESTORE(float, SPHIP_INT8);
        else SPHIP_RESTORE(float, SPHIP_E4M3);
    }
#undef SPHIP_RESTORE
    SPHIP_CHECK_LAUNCH("checkpoint8_restore");
    return SPHIP_OK;
}
