// Shared by the kernels of the dense product (linear.hip, linear_few.hip, linear64.hip, linear128.hip, linear256.hip).
#pragma once
#include "codes8.hpp"
#include "epilogue.hpp"

namespace sphip {

// how element (row, k) of an operand of C[n, m] = sum_k A(n, k) B(m, k) is found
enum { OP_ROWS = 0,      // p[row * ld + k]
       OP_COLS = 1 };    // p[k * ld + row]

struct Operand {
    const void* p;
    int64_t ld;
    int rows;
};

// Whether LDS-DMA can fetch an operand's rows where they are: offsets that fit a tile's buffer descriptor (2^31 bytes: 256 rows
// of bf16, 128 of fp32), bf16 from multiples of 16 bytes. Others are copied first. fp32 elements may lie anywhere: where rows
// are not aligned16 they go 4 bytes at a time.
constexpr int64_t MAX_LD = 1ll << 22;
static inline bool aligned16(const void* p, int64_t ld, int es) { return ((uintptr_t)p & 15) == 0 && ld * es % 16 == 0; }
static inline bool fetchable(const void* p, int64_t ld, int es) { return ld < MAX_LD && (es == 4 || aligned16(p, ld, es)); }

// hipFuncAttributeMaxDynamicSharedMemorySize of a kernel, set once per device (`done`: a bit per device, one word a kernel)
static inline bool reserve_lds(const void* kernel, int bytes, uint64_t& done) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev > 63) return false;
    if (__atomic_load_n(&done, __ATOMIC_RELAXED) >> dev & 1) return true;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) {
        (void)hipGetLastError();
        return false;
    }
    __atomic_fetch_or(&done, 1ull << dev, __ATOMIC_RELAXED);
    return true;
}

struct TileGrid {
    int tilesM, tilesN, splits, steps_per;      // steps_per: K steps of one split
    float* part;                                // [splits][N][Mp] fp32 partial sums, Mp = M rounded up to 4; splits > 1
};

// workgroup -> (split, n tile, m tile): each XCD (workgroup id mod 8, the order the hardware deals them out in) walks a
// contiguous range of bands 8 tiles tall, so that the tiles it runs at a time share their operands in its L2
__device__ __forceinline__ void tile_of(const TileGrid& g, unsigned& split, int& tm, int& tn) {
    const unsigned nb = gridDim.x, xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
    const unsigned q8 = nb >> 3, r8 = nb & 7;
    const unsigned L = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + slot;
    const unsigned tiles = (unsigned)g.tilesM * (unsigned)g.tilesN;
    split = L / tiles;
    const unsigned Lt = L % tiles, band = 8u * (unsigned)g.tilesN, gi = Lt / band, within = Lt % band;
    const unsigned gsize = min((unsigned)g.tilesM - gi * 8, 8u);
    tm = (int)(gi * 8 + within % gsize);
    tn = (int)(within / gsize);
}

typedef __bf16 b16x8_t __attribute__((ext_vector_type(8)));
typedef float acc4_t __attribute__((ext_vector_type(4)));
typedef unsigned w4_t __attribute__((ext_vector_type(4)));
typedef unsigned w2_t __attribute__((ext_vector_type(2)));
typedef void __attribute__((address_space(3)))* lds_t;

// The tail the product's kernels share: ROWS x COLS values of C that a wave has put into its own LDS area [row][out_row(COLS)
// bytes], row r being n = n0 + r, leave so that COLS / 4 lanes store COLS consecutive m of a row. A lane keeps its m: one bias
// load.
// The activation and the 8-bit codes of z are rolled loops over LDS, not unrolled with the rest: inlined per output quad
// they made kernels of 60 to 90 KB, more than the instruction cache holds. Residual and result bypass L2, which holds the
// operands.
constexpr int out_row(int cols) { return cols * 4 + 16; }
constexpr int OUT_ROW = out_row(64);

// The lane's residual pieces and its 4 of the bias, raw, all in flight before the first is used: little else hides their
// latency. No branch and no arithmetic between the loads (either would wait for them one by one): rows past the end load the
// last row again, columns past the end the last column. BIAS false: the bias stays where it is until the end (256 x 256 tiles,
// which load all of this after the product: 16384 x 768 x 3584 91 us against 96).
template <int ROWS, int COLS = 64, bool BIAS = true> struct Residual {
    static constexpr int LANES = COLS / 4, STEP = 64 / LANES, P = ROWS / STEP;     // lanes of a row, rows of a piece, pieces
    w4_t v[P], b;
    __device__ __forceinline__ void load(const Epilogue& epi, const TileGrid& g, int n0, int m0, int N, int M, int lane) {
        const int m = m0 + lane % LANES * 4, nb = n0 + lane / LANES, cols = M - m;
        if (g.splits > 1 || cols <= 0) return;
        if (BIAS && epi.bias != nullptr) {
            const int c1 = min(1, cols - 1), c2 = min(2, cols - 1), c3 = min(3, cols - 1);
            if (epi.bias_dt == SPHIP_F32) {
                const unsigned* p = (const unsigned*)epi.bias + m;
                b = (w4_t){p[0], p[c1], p[c2], p[c3]};
            } else {
                const bf16_t* p = (const bf16_t*)epi.bias + m;
                b = (w4_t){p[0], p[c1], p[c2], p[c3]};
            }
        }
        if (epi.res == nullptr) return;
        if (cols >= 4) {
            if (epi.res_dt == SPHIP_F32) {
#pragma unroll
                for (int i = 0; i < P; ++i)
                    v[i] = __builtin_nontemporal_load((const u4_any*)((const float*)epi.res + (int64_t)min(nb + STEP * i, N - 1) * epi.ldr + m));
            } else {
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const u2_any r = __builtin_nontemporal_load((const u2_any*)((const bf16_t*)epi.res + (int64_t)min(nb + STEP * i, N - 1) * epi.ldr + m));
                    v[i].x = r.x, v[i].y = r.y;
                }
            }
        } else if (epi.res_dt == SPHIP_F32) {      // the row's last, partial piece: missing columns load the last one again
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const unsigned* p = (const unsigned*)epi.res + (int64_t)min(nb + STEP * i, N - 1) * epi.ldr + m;
                v[i].x = p[0], v[i].y = p[min(1, cols - 1)], v[i].z = p[cols - 1];
            }
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const bf16_t* p = (const bf16_t*)epi.res + (int64_t)min(nb + STEP * i, N - 1) * epi.ldr + m;
                v[i].x = p[0], v[i].y = p[min(1, cols - 1)], v[i].z = p[cols - 1];
            }
        }
    }
    __device__ __forceinline__ void get(const Epilogue& epi, int i, int cols, float (&r)[4]) const {
        if (epi.res_dt == SPHIP_F32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = __uint_as_float(v[i][j]);
        } else if (cols >= 4) {
            r[0] = __uint_as_float(v[i].x << 16), r[1] = __uint_as_float(v[i].x & 0xffff0000u);
            r[2] = __uint_as_float(v[i].y << 16), r[3] = __uint_as_float(v[i].y & 0xffff0000u);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = __uint_as_float(v[i][j] << 16);
        }
    }
};

// z + bias of 32 staged rows (a group of the checkpoint) into 8-bit codes: the maxima of a lane's 4 columns over its rows,
// then over the lanes that share them; padding rows and columns get zero codes
template <int FMT, int COLS>
__device__ __forceinline__ void store_codes(const char* mine, const Epilogue& epi, int nb, int m, int N, int M, const float (&bias)[4], int lane) {
    constexpr int LANES = COLS / 4, STEP = 64 / LANES, P = 32 / STEP;
    float v[P][4];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const float4 c = *reinterpret_cast<const float4*>(mine + i * STEP * out_row(COLS));
        const bool in = nb + STEP * i < N;
        v[i][0] = in && m < M ? c.x + bias[0] : 0.f, v[i][1] = in && m + 1 < M ? c.y + bias[1] : 0.f;
        v[i][2] = in && m + 2 < M ? c.z + bias[2] : 0.f, v[i][3] = in && m + 3 < M ? c.w + bias[3] : 0.f;
    }
    float inv[4];
    unsigned scales = 0, bad = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < P; ++i) top = max(top, __float_as_uint(v[i][j]) & 0x7fffffffu);
#pragma unroll
        for (int o = LANES; o < 64; o *= 2) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
        const unsigned b = scale_byte<FMT>(top);
        scales |= b << (8 * j);
        bad |= b == 255u ? 0xffu << (8 * j) : 0u;
        inv[j] = inverse_scale(b);
    }
    if (m >= epi.ldz || nb - lane / LANES >= N) return;
    if (lane < LANES) *reinterpret_cast<unsigned*>(epi.z_scales + (int64_t)(nb >> 5) * epi.ldz + m) = scales;
    const bool keep = epi.act == SPHIP_ACT_RELU;
#pragma unroll
    for (int i = 0; i < P; ++i)
        *reinterpret_cast<unsigned*>((uint8_t*)epi.z + (int64_t)(nb + STEP * i) * epi.ldz + m) = codes_of<FMT>(v[i], inv, keep, bad);
}

template <int ROWS, int COLS, bool BIAS>
__device__ __forceinline__ void finish_rows(char* stage, const Epilogue& epi, const TileGrid& g, unsigned split, int n0, int m0,
                                            int N, int M, int lane, const Residual<ROWS, COLS, BIAS>& res) {
    constexpr int LANES = COLS / 4, STEP = 64 / LANES, P = ROWS / STEP, PITCH = out_row(COLS);
    const int Mp = (M + 3) & ~3;
    const int m = m0 + lane % LANES * 4, nb = n0 + lane / LANES, cols = M - m;
    char* const mine = stage + lane / LANES * PITCH + lane % LANES * 16;           // piece i is STEP rows of PITCH further on
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (g.splits > 1) {
#pragma unroll 4
        for (int i = 0; i < P; ++i)
            if (nb + STEP * i < N && cols > 0)
                *reinterpret_cast<float4*>(g.part + ((int64_t)split * N + nb + STEP * i) * Mp + m) =
                    *reinterpret_cast<const float4*>(mine + i * STEP * PITCH);
    } else {
        float bias[4] = {0.f, 0.f, 0.f, 0.f};
        if (!BIAS && epi.bias != nullptr) {
            if (cols >= 4) load4_as_f32(epi.bias, epi.bias_dt, m, bias);
            else
#pragma unroll
                for (int j = 0; j < 3; ++j)
                    if (j < cols) bias[j] = load_as_f32(epi.bias, epi.bias_dt, m + j);
        }
        if (BIAS && epi.bias != nullptr && cols > 0)
#pragma unroll
            for (int j = 0; j < 4; ++j) bias[j] = __uint_as_float(epi.bias_dt == SPHIP_F32 ? res.b[j] : res.b[j] << 16);
        if (epi.z_scales != nullptr) {                          // (the whole wave: lanes exchange maxima)
#pragma unroll 1
            for (int h = 0; h < ROWS; h += 32) {
                if (epi.z_dt == SPHIP_INT8) store_codes<SPHIP_INT8, COLS>(mine + h * PITCH, epi, nb + h, m, N, M, bias, lane);
                else store_codes<SPHIP_E4M3, COLS>(mine + h * PITCH, epi, nb + h, m, N, M, bias, lane);
            }
        }
        if (epi.bias != nullptr || epi.act != SPHIP_ACT_NONE || epi.z != nullptr) {
            const bool values = epi.z != nullptr && epi.z_scales == nullptr;
#pragma unroll 2
            for (int i = 0; i < P; ++i) {
                const int n = nb + STEP * i;
                float4* at = reinterpret_cast<float4*>(mine + i * STEP * PITCH);
                const float4 c = *at;
                float v[4] = {c.x + bias[0], c.y + bias[1], c.z + bias[2], c.w + bias[3]};
                if (values && n < N) {
                    if (cols >= 4) store4_stream(epi.z, epi.z_dt, n * epi.ldz + m, v);
                    else
#pragma unroll
                        for (int j = 0; j < 3; ++j)
                            if (j < cols) store_from_f32(epi.z, epi.z_dt, n * epi.ldz + m + j, v[j]);
                }
                act_value4(v, epi.act);
                *at = make_float4(v[0], v[1], v[2], v[3]);
            }
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int n = nb + STEP * i;
            if (n >= N) continue;
            const float4 c = *reinterpret_cast<const float4*>(mine + i * STEP * PITCH);
            float v[4] = {c.x, c.y, c.z, c.w};
            if (epi.res != nullptr) {
                float r[4];
                res.get(epi, i, cols, r);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += r[j];
            }
            if (cols >= 4) {
                store4_stream(epi.out, epi.out_dt, n * epi.ldo + m, v);
            } else {
#pragma unroll
                for (int j = 0; j < 3; ++j)
                    if (j < cols) store_from_f32(epi.out, epi.out_dt, n * epi.ldo + m + j, v[j]);
            }
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// checkpoint8.hip: x (N, D) in 8 bits; with `packed` also a copy of it in rows of ldp elements, zeros behind column D
int save_codes(const char* what, const void* x, int dtype, int64_t ldx, int fmt, int keep_sign, uint8_t* codes, uint8_t* scales,
               int64_t ldq, void* packed, int64_t ldp, int64_t N, int64_t D, hipStream_t s);

// linear_few.hip: the whole product for N <= 64, x and W contiguous in K (no codes of z)
constexpr int FEW = 64;
int launch_linear_few(const char* what, int dtype, const Operand& X, const Operand& W, const Epilogue& epi, int64_t K, hipStream_t s);

// The tiled kernels (256: bf16 only): how they split K, their launch (the caller joins). Operands: fetchable(), in bf16 and
// with 16 of `bytes` K whole 16-byte pieces where it is the contiguous index.
// KB: rows of an OP_COLS B, which may be fewer than K (whole 16-byte pieces where A is OP_ROWS): B counts as zero from there.
int launch_linear256(const char* what, int mode_a, int mode_b, const Operand& A, const Operand& B, const Epilogue& epi, int64_t K,
                     int64_t KB, const TileGrid& g, hipStream_t s);
int linear64_splits(int dtype, int64_t N, int64_t M, int64_t K);
int launch_linear64(const char* what, int dtype, int bytes, int mode_a, int mode_b, const Operand& A, const Operand& B,
                    const Epilogue& epi, int64_t K, int64_t KB, const TileGrid& g, hipStream_t s);
int linear128_splits(int dtype, int64_t N, int64_t M, int64_t K);
int launch_linear128(const char* what, int dtype, int bytes, int mode_a, int mode_b, const Operand& A, const Operand& B,
                     const Epilogue& epi, int64_t K, int64_t KB, const TileGrid& g, hipStream_t s);

}  // namespace sphip
