// The dense product's kernel for large bf16 shapes: C[n, m] = sum_k A(n, k) B(m, k), a 256 x 256 tile of C per workgroup of
// 8 waves (2 groups of m x 4 of n, 128 x 64 outputs per wave), 64 of K per step, v_mfma_f32_16x16x32_bf16.
//
// Schedule: that of encoder_gemm256.hip. Operand tiles arrive by LDS-DMA into a double-buffered 128 KiB image; the two wave
// groups sharing a SIMD run staggered by one barrier, one reading fragments (L segments) while the other multiplies (M):
//     L0: read A(t), B-lo(t)     | B-hi(t) landed             M0: DMA B-hi(t+1)          | 32 MFMA
//     L1: read B-hi(t)           | A(t+1), B-lo(t+1) landed   M1: DMA A(t+2), B-lo(t+2)  | 32 MFMA
// A region read in segment r was awaited two segments before (so every wave has passed a barrier since) and is overwritten
// by DMA issued at the earliest in segment r + 3.
//
// An operand is either contiguous in K (OP_ROWS: image [row][8 chunks of 8 k], chunk XOR (row >> 1) & 7, ds_read_b128) or
// contiguous in its rows (OP_COLS: the gradient products). The latter is not transposed in memory: its image is [k][chunks
// of 8 rows] as it comes, and ds_read_b64_tr_b16 hands every lane 4 consecutive k of its row (of 16 lanes, lane i names
// k = i / 4 and rows 4 (i % 4) .. + 3 and receives row i). Chunk XOR 2 ((k & 3) + 4 ((k >> 3) & 1)) spreads the 4 k of one
// read, and the 8 apart ones of the neighbouring 16 lanes, over 8 different 32-byte slots: no bank conflicts.
// LDS-DMA writes linearly, so both swizzles are applied to the per-lane source address; rows and K past the end read as
// zeros by the buffer descriptors' range check (K past the end of an OP_ROWS operand does not, hence K % 64 == 0 there).
#include "linear.hpp"

namespace sphip {

typedef __bf16 b16x8_t __attribute__((ext_vector_type(8)));
typedef float acc4_t __attribute__((ext_vector_type(4)));
typedef unsigned w4_t __attribute__((ext_vector_type(4)));
typedef unsigned w2_t __attribute__((ext_vector_type(2)));
typedef void __attribute__((address_space(3)))* lds_t;

constexpr int T256 = 256, K64 = 64;
constexpr int RG_A = 0, RG_BLO = 32768, RG_BHI = 49152, IMG = 65536;
constexpr int OUT_ROW = 272;                       // epilogue staging: 64 fp32 + 16 bytes per row of C
constexpr int OUT_WAVE = 64 * OUT_ROW;
constexpr int LDS256 = (2 * IMG > 8 * OUT_WAVE) ? 2 * IMG : 8 * OUT_WAVE;

__device__ __forceinline__ void segment_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}

#define LIN_VMCNT(n) asm volatile("s_waitcnt vmcnt(" #n ")" ::: "memory")

// Four 16-row fragments of 64 k: [tile][32-k step]. Reads are issued from inline asm (the compiler would drain the DMA
// queue before each visible LDS read), completed by wait(), which names every destination register.
template <int MODE> struct Frag;
template <> struct Frag<OP_ROWS> {
    w4_t v[4][2];
    // a0 / a1: the lane's addresses for the two 32-k steps; tiles are 16 rows = 2048 bytes apart
    __device__ __forceinline__ void read(const unsigned (&a)[4], unsigned bo, int region) {
#define LIN_DSR(i, ks) \
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v[i][ks]) : "v"(a[ks] + bo + region), "i"((i) * 2048))
        LIN_DSR(0, 0); LIN_DSR(0, 1); LIN_DSR(1, 0); LIN_DSR(1, 1);
        LIN_DSR(2, 0); LIN_DSR(2, 1); LIN_DSR(3, 0); LIN_DSR(3, 1);
#undef LIN_DSR
    }
    __device__ __forceinline__ void wait() {
        asm volatile("s_waitcnt lgkmcnt(0)"
                     : "+v"(v[0][0]), "+v"(v[0][1]), "+v"(v[1][0]), "+v"(v[1][1]), "+v"(v[2][0]), "+v"(v[2][1]), "+v"(v[3][0]),
                       "+v"(v[3][1]));
    }
    __device__ __forceinline__ b16x8_t get(int i, int ks) const { return __builtin_bit_cast(b16x8_t, v[i][ks]); }
    // per-lane addresses: rows of the wave start at row0 of the region
    static __device__ __forceinline__ void addresses(unsigned lds0, int row0, int lane, unsigned (&a)[4]) {
        const int r16 = lane & 15, q4 = lane >> 4;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) a[ks] = lds0 + (row0 + r16) * 128 + (((4 * ks + q4) ^ ((r16 >> 1) & 7)) << 4);
        a[2] = a[3] = 0;
    }
};
template <> struct Frag<OP_COLS> {
    w2_t v[4][2][2];                                   // [tile][32-k step][4-k half]
    // a[i]: the lane's address in tile i; PITCH bytes per k row (512 for A, 256 for a half of B)
    template <int PITCH> __device__ __forceinline__ void read_p(const unsigned (&a)[4], unsigned bo, int region) {
#define LIN_DSR(i, ks, h)                                                                                        \
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2"                                                           \
                 : "=v"(v[i][ks][h])                                                                             \
                 : "v"(a[i] + bo + region), "i"((ks) * 32 * PITCH + (h) * 4 * PITCH))
        LIN_DSR(0, 0, 0); LIN_DSR(0, 0, 1); LIN_DSR(0, 1, 0); LIN_DSR(0, 1, 1);
        LIN_DSR(1, 0, 0); LIN_DSR(1, 0, 1); LIN_DSR(1, 1, 0); LIN_DSR(1, 1, 1);
        LIN_DSR(2, 0, 0); LIN_DSR(2, 0, 1); LIN_DSR(2, 1, 0); LIN_DSR(2, 1, 1);
        LIN_DSR(3, 0, 0); LIN_DSR(3, 0, 1); LIN_DSR(3, 1, 0); LIN_DSR(3, 1, 1);
#undef LIN_DSR
    }
    __device__ __forceinline__ void wait() {
        asm volatile("s_waitcnt lgkmcnt(0)"
                     : "+v"(v[0][0][0]), "+v"(v[0][0][1]), "+v"(v[0][1][0]), "+v"(v[0][1][1]), "+v"(v[1][0][0]), "+v"(v[1][0][1]),
                       "+v"(v[1][1][0]), "+v"(v[1][1][1]), "+v"(v[2][0][0]), "+v"(v[2][0][1]), "+v"(v[2][1][0]),
                       "+v"(v[2][1][1]), "+v"(v[3][0][0]), "+v"(v[3][0][1]), "+v"(v[3][1][0]), "+v"(v[3][1][1]));
    }
    __device__ __forceinline__ b16x8_t get(int i, int ks) const {
        const w4_t w = __builtin_shufflevector(v[i][ks][0], v[i][ks][1], 0, 1, 2, 3);
        return __builtin_bit_cast(b16x8_t, w);
    }
    static __device__ __forceinline__ void addresses(unsigned lds0, int chunk0, int pitch, int lane, unsigned (&a)[4]) {
        const int r16 = lane & 15, q4 = lane >> 4;
        const int k = 8 * q4 + (r16 >> 2), f = (k & 3) + 4 * ((k >> 3) & 1);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            a[i] = lds0 + k * pitch + (((chunk0 + 2 * i + ((r16 & 3) >> 1)) ^ (2 * f)) << 4) + (r16 & 1) * 8;
    }
};

// One operand of the kernel: descriptor, per-lane source offset, DMA pieces. Which = 0: A (one region of 256 rows, 4 pieces
// per K step), 1: B (regions lo / hi of 128 rows, 2 pieces each: rows [0,64) and [64,128) of both 128-row wave groups).
template <int MODE, int WHICH> struct Source {
    __amdgpu_buffer_rsrc_t rsrc;
    unsigned voff, piece, step;            // bytes: lane offset, between pieces, between K steps
    __device__ __forceinline__ void init(const Operand& o, int row0, int64_t k0, int64_t K, int tid) {
        const bf16_t* p = (const bf16_t*)o.p;
        const unsigned ld2 = (unsigned)o.ld * 2u;
        if (MODE == OP_ROWS) {
            const int hr = tid >> 3, ch = (tid & 7) ^ ((hr >> 1) & 7);
            const int rows = min(T256, o.rows - row0);
            rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(p + (int64_t)row0 * o.ld + k0), 0,
                                                     (int)((unsigned)(rows - 1) * ld2 + (unsigned)(K - k0) * 2u), 0x00020000);
            voff = (unsigned)hr * ld2 + (unsigned)ch * 16u;
            piece = 64u * ld2;
            step = K64 * 2;
        } else {
            constexpr int LOG = WHICH == 0 ? 5 : 4;    // chunks per k row: 32 (A), 16 (a half of B)
            const int kr = tid >> LOG, f = (kr & 3) + 4 * ((kr >> 3) & 1);
            const int c = (tid & ((1 << LOG) - 1)) ^ (2 * f);
            const int col = WHICH == 0 ? c * 8 : (c >> 3) * 128 + (c & 7) * 8;
            // (the end rounded up to a piece: a dword that crosses the end reads as zero, with it the last of an odd number
            // of rows; rows are 16-byte aligned, so the piece is the one that holds the last element)
            rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(p + k0 * o.ld + row0), 0,
                                                     (int)(K > k0 ? (unsigned)(K - 1 - k0) * ld2 + ((unsigned)(o.rows - row0) * 2u + 15u) / 16u * 16u : 0u),
                                                     0x00020000);
            voff = (unsigned)kr * ld2 + (unsigned)col * 2u;
            piece = (512u >> LOG) * ld2;
            step = K64 * ld2;
        }
    }
    // piece i of K step t; hi: the second half of B
    __device__ __forceinline__ void dma(char* lds, int t, int i, int hi) const {
        unsigned so = (unsigned)t * step;
        if (MODE == OP_ROWS) so += (unsigned)(WHICH == 0 ? i : 2 * i + hi) * piece;
        else so += (unsigned)i * piece + (WHICH == 1 ? (unsigned)hi * 128u : 0u);
        // the whole offset in the register the range check looks at
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_t)lds, 16, voff + so, 0, 0, 0);
    }
};

template <int MA, int MB>
__global__ __launch_bounds__(512, 2) void linear256_kernel(Operand A, Operand B, Epilogue epi, int64_t K, int64_t KB, TileGrid g) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    unsigned split;
    int tm, tn;
    tile_of(g, split, tm, tn);
    const int m0 = tm * T256, n0 = tn * T256;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3, r16 = lane & 15, q4 = lane >> 4;
    const int64_t k0 = (int64_t)split * g.steps_per * K64;
    const int steps = (int)min((int64_t)g.steps_per, (K - k0 + K64 - 1) / K64);

    Source<MA, 0> sa;
    Source<MB, 1> sb;
    sa.init(A, n0, k0, K, tid);
    sb.init(B, m0, k0, KB, tid);
    char* const dst = smem + wave * 1024;              // wave-uniform base of a 1 KiB piece
    auto dma_a = [&](int t, int i) { sa.dma(dst + (t & 1) * IMG + RG_A + 8192 * i, t, i, 0); };
    auto dma_b = [&](int hi, int t, int i) { sb.dma(dst + (t & 1) * IMG + (hi ? RG_BHI : RG_BLO) + 8192 * i, t, i, hi); };

    const unsigned lds0 = (unsigned)(size_t)(lds_t)smem;
    unsigned aa[4], ab[4];
    if constexpr (MA == OP_ROWS) Frag<MA>::addresses(lds0, wn * 64, lane, aa);
    else Frag<MA>::addresses(lds0, wn * 8, 512, lane, aa);
    if constexpr (MB == OP_ROWS) Frag<MB>::addresses(lds0, wm * 64, lane, ab);
    else Frag<MB>::addresses(lds0, wm * 8, 256, lane, ab);
    Frag<MA> fa;
    Frag<MB> fb;
    auto read_a = [&](unsigned bo) {
        if constexpr (MA == OP_ROWS) fa.read(aa, bo, RG_A);
        else fa.template read_p<512>(aa, bo, RG_A);
    };
    auto read_b = [&](unsigned bo, int region) {
        if constexpr (MB == OP_ROWS) fb.read(ab, bo, region);
        else fb.template read_p<256>(ab, bo, region);
    };

    acc4_t acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = (acc4_t){0.f, 0.f, 0.f, 0.f};

    // 32 MFMAs of an M segment, its DMA issues spread between them, the closing barrier raised one group early (its release
    // latency then hides under the last MFMAs)
    auto multiply = [&](int mbase, int ndma, auto dma) {
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
                for (int nt = 0; nt < 4; ++nt)
                    acc[mbase + mt][nt] =
                        __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb.get(mt, ks), fa.get(nt, ks), acc[mbase + mt][nt], 0, 0, 0);
                const int j = ks * 4 + mt;
                if (j < ndma) {
                    __builtin_amdgcn_sched_barrier(0);
                    dma(j);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (j == 6) segment_barrier();
            }
        __builtin_amdgcn_s_setprio(0);
    };

#pragma unroll
    for (int i = 0; i < 4; ++i) dma_a(0, i);
    dma_b(0, 0, 0), dma_b(0, 0, 1), dma_b(1, 0, 0), dma_b(1, 0, 1);
    if (steps > 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) dma_a(1, i);
        dma_b(0, 1, 0), dma_b(0, 1, 1);
        LIN_VMCNT(8);
    } else {
        LIN_VMCNT(2);
    }
    segment_barrier();
    if (wm == 1) segment_barrier();

    // outstanding DMA per wave, in issue order, at the two waits:
    //   L0: [B-hi(t) 2][A(t+1) 4][B-lo(t+1) 2]      L1: [A(t+1) 4][B-lo(t+1) 2][B-hi(t+1) 2]
#define LIN_STEP(ISSUE_HI, ISSUE_A, WAIT_L0, WAIT_L1)                                              \
    {                                                                                             \
        const unsigned bo = (unsigned)(t & 1) * IMG;                                              \
        read_a(bo);                                                                               \
        read_b(bo, RG_BLO);                                                                       \
        WAIT_L0;                                                                                  \
        segment_barrier();                                                                        \
        fa.wait();                                                                                \
        fb.wait();                                                                                \
        multiply(0, (ISSUE_HI) ? 2 : 0, [&](int j) { dma_b(1, t + 1, j); });                      \
        read_b(bo, RG_BHI);                                                                       \
        WAIT_L1;                                                                                  \
        segment_barrier();                                                                        \
        fb.wait();                                                                                \
        multiply(4, (ISSUE_A) ? 6 : 0, [&](int j) {                                               \
            if (j < 4) dma_a(t + 2, j);                                                           \
            else dma_b(0, t + 2, j - 4);                                                          \
        });                                                                                       \
    }
    int t = 0;
    for (; t < steps - 2; ++t) LIN_STEP(true, true, LIN_VMCNT(6), LIN_VMCNT(2))
    if (steps > 1) {
        LIN_STEP(true, false, LIN_VMCNT(6), LIN_VMCNT(2))
        ++t;
    }
    LIN_STEP(false, false, LIN_VMCNT(0), (void)0)
#undef LIN_STEP
    if (wm == 0) segment_barrier();          // matches the stagger barrier of the other group

    // ---- epilogue. A lane holds 4 consecutive m of one n per accumulator; each wave turns its 64 x 128 part in two halves
    // of 64 x 64 through a private LDS area (the operand image is dead), so that 16 lanes store 64 consecutive m of a row
    // and a lane keeps its m: one bias load per half. The half's 16 residual pieces are all in flight before the first is
    // used (one workgroup runs per compute unit: nothing else hides their latency). Residual and result bypass L2, which
    // holds the operands.
    const int N = A.rows, M = B.rows, Mp = (M + 3) & ~3;
    char* const stage = smem + wave * OUT_WAVE;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int m = m0 + wm * 128 + half * 64 + r16 * 4, nb = n0 + wn * 64 + q4;
        const bool whole = g.splits == 1 && epi.vec && m + 3 < M;
        w4_t res[16];
        float bias[4] = {0.f, 0.f, 0.f, 0.f};
        if (whole && epi.res != nullptr) {
            if (epi.res_dt == SPHIP_F32) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (nb + 4 * i < N)
                        res[i] = __builtin_nontemporal_load((const w4_t*)((const float*)epi.res + (int64_t)(nb + 4 * i) * epi.ldr + m));
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (nb + 4 * i < N) {
                        const w2_t r = __builtin_nontemporal_load((const w2_t*)((const bf16_t*)epi.res + (int64_t)(nb + 4 * i) * epi.ldr + m));
                        res[i] = (w4_t){r.x << 16, r.x & 0xffff0000u, r.y << 16, r.y & 0xffff0000u};
                    }
            }
        }
        if (whole && epi.bias != nullptr) load4_as_f32(epi.bias, epi.bias_dt, m, bias);
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
                *reinterpret_cast<acc4_t*>(stage + (nt * 16 + r16) * OUT_ROW + (mt * 16 + q4 * 4) * 4) = acc[half * 4 + mt][nt];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (whole) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int n = nb + 4 * i;
                if (n >= N) continue;
                const float4 c = *reinterpret_cast<const float4*>(stage + (i * 4 + q4) * OUT_ROW + r16 * 16);
                float v[4] = {c.x + bias[0], c.y + bias[1], c.z + bias[2], c.w + bias[3]};
                if (epi.z != nullptr) store4_from_f32(epi.z, epi.z_dt, n * epi.ldz + m, v);
                if (epi.act != SPHIP_ACT_NONE) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = act_value(v[j], epi.act);
                }
                if (epi.res != nullptr) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] += __uint_as_float(res[i][j]);
                }
                if (epi.out_dt == SPHIP_F32) {
                    const acc4_t o = {v[0], v[1], v[2], v[3]};
                    __builtin_nontemporal_store(o, (acc4_t*)((float*)epi.out + n * epi.ldo + m));
                } else {
                    const w2_t o = {(unsigned)f32_to_bf16(v[0]) | ((unsigned)f32_to_bf16(v[1]) << 16),
                                    (unsigned)f32_to_bf16(v[2]) | ((unsigned)f32_to_bf16(v[3]) << 16)};
                    __builtin_nontemporal_store(o, (w2_t*)((bf16_t*)epi.out + n * epi.ldo + m));
                }
            }
        } else if (m < M) {
#pragma unroll 4
            for (int i = 0; i < 16; ++i) {
                const int n = nb + 4 * i;
                if (n >= N) continue;
                const float4 c = *reinterpret_cast<const float4*>(stage + (i * 4 + q4) * OUT_ROW + r16 * 16);
                float v[4] = {c.x, c.y, c.z, c.w};
                if (g.splits > 1) *reinterpret_cast<float4*>(g.part + ((int64_t)split * N + n) * Mp + m) = c;
                else epilogue4(epi, n, m, M, v);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

static bool dma_ok(int mode, const Operand& o, int64_t K) {
    if (((uintptr_t)o.p & 15) != 0 || o.ld % 8 != 0) return false;
    // 32-bit byte offsets inside a tile's descriptor, over the whole K range
    if (mode == OP_ROWS) return K % K64 == 0 && o.ld * 2 * T256 + K * 2 < (1ll << 31);
    return mode == OP_COLS && (K + K64) * o.ld * 2 < (1ll << 31);
}

bool linear256_takes(int mode_a, int mode_b, const Operand& A, const Operand& B, int64_t K) {
    return dma_ok(mode_a, A, K) && dma_ok(mode_b, B, K);
}

// Splits of the K range: as many as still give each of the 256 compute units one workgroup, 8 steps each at least.
int linear256_splits(int64_t N, int64_t M, int64_t K) {
    const int64_t tiles = cdiv(N, T256) * cdiv(M, T256), steps = cdiv(K, K64);
    int64_t s = 256 / tiles;
    if (s > steps / 8) s = steps / 8;
    return s < 1 ? 1 : (int)s;
}

int launch_linear256(const char* what, int mode_a, int mode_b, const Operand& A, const Operand& B, const Epilogue& epi, int64_t K,
                     int64_t KB, const TileGrid& g, hipStream_t s) {
    typedef void (*kern_t)(Operand, Operand, Epilogue, int64_t, int64_t, TileGrid);
    const int which = mode_a == OP_ROWS ? (mode_b == OP_ROWS ? 0 : 1) : 2;
    static const kern_t kerns[3] = {linear256_kernel<OP_ROWS, OP_ROWS>, linear256_kernel<OP_ROWS, OP_COLS>,
                                    linear256_kernel<OP_COLS, OP_COLS>};
    SPHIP_REQUIRE(hipFuncSetAttribute((const void*)kerns[which], hipFuncAttributeMaxDynamicSharedMemorySize, LDS256) == hipSuccess,
                  SPHIP_ELAUNCH, "%s: cannot reserve %d bytes of LDS", what, LDS256);
    const int64_t blocks = (int64_t)g.tilesM * g.tilesN * g.splits;
    hipLaunchKernelGGL(kerns[which], dim3((unsigned)blocks), dim3(512), LDS256, s, A, B, epi, K, KB, g);
    SPHIP_CHECK_LAUNCH(what);
    return SPHIP_OK;
}

}  // namespace sphip
