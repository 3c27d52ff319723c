// The dense product for a few tokens (N <= 64): y = act(x W^T + b) + r, one launch.
//
// Bound: reading W once (M D elements; 4096 x 4096 bf16: 32 MiB, 6.5 us at the 5.15 TB/s a large copy reaches; one token
// takes 7.6). So W goes from memory straight into MFMA operands, nothing staged: a workgroup owns 16 or 32 rows of W, its 8 waves
// take turns at pieces of K (consecutive waves read consecutive pieces of a row), each lane 16 bytes of one row per
// instruction, the next pieces requested before the present ones are multiplied. x is read through the caches by every
// workgroup, as the MFMA's other operand (rows past N repeat the last one; their results are dropped). The 8 partial sums
// meet in LDS and are added in order.
// Any stride and element alignment: the loads are unaligned vectors, only the last piece of a row takes element loads.
#include "linear.hpp"

namespace sphip {

template <typename T> struct Piece;                          // 16 bytes of K of one row
template <> struct Piece<bf16_t> {
    static constexpr int E = 8, K = 32;                      // elements per lane, K per MFMA group (4 lanes' pieces)
    static __device__ __forceinline__ acc4_t mma(const w4_t& a, const w4_t& b, acc4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8_t, a), __builtin_bit_cast(b16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ w4_t tail(const bf16_t* p, int n) {
        w4_t r = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 7; ++j)
            if (j < n) r[j >> 1] |= (unsigned)p[j] << ((j & 1) * 16);
        return r;
    }
};
template <> struct Piece<float> {
    static constexpr int E = 4, K = 16;
    static __device__ __forceinline__ acc4_t mma(const w4_t& a, const w4_t& b, acc4_t c) {
        // four 4-wide MFMAs: element j of the lanes' pieces each time; both operands agree on which K that is
#pragma unroll
        for (int j = 0; j < 4; ++j)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ w4_t tail(const float* p, int n) {
        w4_t r = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (j < n) r[j] = __float_as_uint(p[j]);
        return r;
    }
};

constexpr int FEW_WAVES = 8;

// NT x MT tiles of 16 tokens x 16 rows of W; U pieces of K per wave and round
template <typename T, int NT, int MT, int U>
__global__ __launch_bounds__(512) void linear_few_kernel(Operand X, Operand W, Epilogue epi, int64_t K) {
    constexpr int E = Piece<T>::E, KG = Piece<T>::K;
    __shared__ acc4_t red[FEW_WAVES][NT * MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, q4 = lane >> 4;
    const int N = X.rows, M = W.rows, m0 = blockIdx.x * (16 * MT);
    const T *w[MT], *x[NT];
#pragma unroll
    for (int j = 0; j < MT; ++j) w[j] = (const T*)W.p + (int64_t)min(m0 + j * 16 + r16, M - 1) * W.ld + q4 * E;
#pragma unroll
    for (int i = 0; i < NT; ++i) x[i] = (const T*)X.p + (int64_t)min(i * 16 + r16, N - 1) * X.ld + q4 * E;

    acc4_t acc[MT][NT];
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[j][i] = (acc4_t){0.f, 0.f, 0.f, 0.f};
    w4_t wa[2][MT][U], xa[2][NT][U];
    // whole rounds: U groups of KG per wave
    const int64_t round = (int64_t)FEW_WAVES * U * KG, rounds = K / round;
    auto load = [&](int b, int64_t k) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < MT; ++j) __builtin_memcpy(&wa[b][j][u], w[j] + k + u * KG, 16);
#pragma unroll
            for (int i = 0; i < NT; ++i) __builtin_memcpy(&xa[b][i][u], x[i] + k + u * KG, 16);
        }
    };
    auto multiply = [&](int b) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < MT; ++j)
#pragma unroll
                for (int i = 0; i < NT; ++i) acc[j][i] = Piece<T>::mma(wa[b][j][u], xa[b][i][u], acc[j][i]);
    };
    const int64_t k0 = (int64_t)wave * U * KG;
    if (rounds > 0) load(0, k0);
    int64_t r = 0;
    for (; r + 2 <= rounds; r += 2) {
        load(1, k0 + (r + 1) * round);
        multiply(0);
        if (r + 2 < rounds) load(0, k0 + (r + 2) * round);
        multiply(1);
    }
    if (r < rounds) multiply(0);
    // the rest, group by group
    for (int64_t k = rounds * round + wave * KG; k < K; k += FEW_WAVES * KG) {
        const int n = (int)min((int64_t)E, K - k - q4 * E);
        w4_t a[MT], b[NT];
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            a[j] = (w4_t){0, 0, 0, 0};
            if (n >= E) __builtin_memcpy(&a[j], w[j] + k, 16);
            else if (n > 0) a[j] = Piece<T>::tail(w[j] + k, n);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            b[i] = (w4_t){0, 0, 0, 0};
            if (n >= E) __builtin_memcpy(&b[i], x[i] + k, 16);
            else if (n > 0) b[i] = Piece<T>::tail(x[i] + k, n);
        }
#pragma unroll
        for (int j = 0; j < MT; ++j)
#pragma unroll
            for (int i = 0; i < NT; ++i) acc[j][i] = Piece<T>::mma(a[j], b[i], acc[j][i]);
    }
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int i = 0; i < NT; ++i) red[wave][j * NT + i][lane] = acc[j][i];
    __syncthreads();
    // a lane of the accumulator layout holds 4 consecutive m of one n
    const int tile = threadIdx.x >> 6;
    if (tile >= NT * MT) return;
    const int n = tile % NT * 16 + r16, m = m0 + tile / NT * 16 + q4 * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < FEW_WAVES; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += red[s][tile][lane][j];
    if (n < N && m < M) epilogue4(epi, n, m, M, v);
}

template <typename T, int MT> static void launch(const Operand& X, const Operand& W, const Epilogue& epi, int64_t K, hipStream_t s) {
    const dim3 grid((unsigned)cdiv(W.rows, 16 * MT)), block(512);
    if (X.rows <= 16) hipLaunchKernelGGL((linear_few_kernel<T, 1, MT, 4>), grid, block, 0, s, X, W, epi, K);
    else if (X.rows <= 32) hipLaunchKernelGGL((linear_few_kernel<T, 2, MT, 4>), grid, block, 0, s, X, W, epi, K);
    else hipLaunchKernelGGL((linear_few_kernel<T, 4, MT, MT == 1 ? 4 : 2>), grid, block, 0, s, X, W, epi, K);
}

// 32 rows of W per workgroup (half the reads of x) where 16 would give a compute unit more than one of them: 24 x 2048 x 6000
// 9.8 us against 13.1, 2048 x 8000 10.1 against 13.5 (fp32 20.7 against 26.2); where they would not, 24 x 2048 x 4096 takes 9.5
// against 7.8. Up to 16 tokens only while 32 rows still are one round, 16 x 2048 x 8000 9.1 against 10.3, 2048 x 8256 14.6 against
// 13.6; up to 8 not at all: one token 4096 x 8000 16.0 against 13.5 (8 tokens: 2048 x 6000 8.0 against 9.2, 4096 x 8000 16.3 / 15.3).
int launch_linear_few(const char* what, int dtype, const Operand& X, const Operand& W, const Epilogue& epi, int64_t K, hipStream_t s) {
    const bool bf = dtype == SPHIP_BF16, wide = W.rows > 4096 && (X.rows > 16 || (X.rows > 8 && W.rows <= 8192));
    if (bf && wide) launch<bf16_t, 2>(X, W, epi, K, s);
    else if (bf) launch<bf16_t, 1>(X, W, epi, K, s);
    else if (wide) launch<float, 2>(X, W, epi, K, s);
    else launch<float, 1>(X, W, epi, K, s);
    SPHIP_CHECK_LAUNCH(what);
    return SPHIP_OK;
}

}  // namespace sphip
