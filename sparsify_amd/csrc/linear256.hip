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
// Images and fragment reads: linear_dma.hpp.
#include "linear_dma.hpp"

namespace sphip {

constexpr int T256 = 256;
constexpr int RG_A = 0, RG_BLO = 32768, RG_BHI = 49152, IMG = 65536;
constexpr int OUT_WAVE = 64 * OUT_ROW;             // epilogue staging per wave
constexpr int LDS256 = (2 * IMG > 8 * OUT_WAVE) ? 2 * IMG : 8 * OUT_WAVE;

__device__ __forceinline__ void segment_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}

// One operand of the kernel: descriptor, per-lane source offset, DMA pieces. Which = 0: A (one region of 256 rows, 4 pieces
// per K step), 1: B (regions lo / hi of 128 rows, 2 pieces each: rows [0,64) and [64,128) of both 128-row wave groups).
template <int MODE, int WHICH> struct Source256 {
    const bf16_t* base;                    // of the tile and the split, uniform
    unsigned ld2, edge;                    // bytes: row stride; OP_ROWS: of the descriptor, OP_COLS: of its last k row
    unsigned voff, piece;                  // bytes: lane offset, between pieces
    int left;                              // OP_ROWS: 16-byte pieces of K from the lane's on; OP_COLS: k rows
    __device__ __forceinline__ void init(const Operand& o, int row0, int64_t k0, int64_t K, int tid) {
        ld2 = (unsigned)o.ld * 2u;
        if (MODE == OP_ROWS) {
            const int hr = tid >> 3, ch = (tid & 7) ^ ((hr >> 1) & 7);
            base = (const bf16_t*)o.p + (int64_t)row0 * o.ld + k0;
            edge = (unsigned)(min(T256, o.rows - row0) - 1) * ld2 + (unsigned)(K - k0) * 2u;
            voff = (unsigned)hr * ld2 + (unsigned)ch * 16u;
            piece = 64u * ld2;
            left = (int)((K - k0) / 8) - ch;
        } else {
            constexpr int LOG = WHICH == 0 ? 5 : 4;    // chunks per k row: 32 (A), 16 (a half of B)
            const int kr = tid >> LOG, f = (kr & 3) + 4 * ((kr >> 3) & 1);
            const int c = (tid & ((1 << LOG) - 1)) ^ (2 * f);
            const int col = WHICH == 0 ? c * 8 : (c >> 3) * 128 + (c & 7) * 8;
            base = (const bf16_t*)o.p + k0 * o.ld + row0;
            edge = ((unsigned)(o.rows - row0) * 2u + 15u) / 16u * 16u;         // (why a whole piece: linear_dma.hpp)
            voff = (unsigned)kr * ld2 + (unsigned)col * 2u;
            piece = (512u >> LOG) * ld2;
            left = (int)(K - k0);
        }
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t step(int t) const {      // (see linear_dma.hpp)
        if (MODE == OP_ROWS) return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)edge, 0x00020000);
        const unsigned rows = (unsigned)min(K64, left - t * K64);
        return __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)base + (uint64_t)((unsigned)t * K64) * ld2), 0,
                                                 (int)((rows - 1) * ld2 + edge), 0x00020000);
    }
    __device__ __forceinline__ void last(int t) {
        if (MODE == OP_ROWS && 8 * t >= left) voff |= PAST_END;
    }
    // piece i of K step t; hi: the second half of B
    __device__ __forceinline__ void dma(char* lds, int t, int i, int hi) const {
        const __amdgpu_buffer_rsrc_t rsrc = step(t);
        unsigned so;
        if (MODE == OP_ROWS) so = (unsigned)t * 128u + (unsigned)(WHICH == 0 ? i : 2 * i + hi) * piece;
        else so = (unsigned)i * piece + (WHICH == 1 ? (unsigned)hi * 128u : 0u);
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
    const int wm = wave >> 2, wn = wave & 3;
    const int64_t k0 = (int64_t)split * g.steps_per * K64;
    const int steps = (int)min((int64_t)g.steps_per, (K - k0 + K64 - 1) / K64);

    Source256<MA, 0> sa;
    Source256<MB, 1> sb;
    sa.init(A, n0, k0, K, tid);
    sb.init(B, m0, k0, KB, tid);
    char* const dst = smem + wave * 1024;              // wave-uniform base of a 1 KiB piece
    auto dma_a = [&](int t, int i) { sa.dma(dst + (t & 1) * IMG + RG_A + 8192 * i, t, i, 0); };
    auto dma_b = [&](int hi, int t, int i) { sb.dma(dst + (t & 1) * IMG + (hi ? RG_BHI : RG_BLO) + 8192 * i, t, i, hi); };

    const unsigned lds0 = (unsigned)(size_t)(lds_t)smem;
    Frag<bf16_t, MA, 512> fa;
    Frag<bf16_t, MB, 256> fb;
    fa.init(lds0, wn * 64, lane);
    fb.init(lds0, wm * 64, lane);
    auto read_a = [&](unsigned bo) {
        fa.template read<0>(bo + RG_A);
        fa.template read<1>(bo + RG_A);
    };
    auto read_b = [&](unsigned bo, int region) {
        fb.template read<0>(bo + region);
        fb.template read<1>(bo + region);
    };
    auto wait_a = [&] { fa.template wait<0, 0>(), fa.template wait<1, 0>(); };
    auto wait_b = [&] { fb.template wait<0, 0>(), fb.template wait<1, 0>(); };

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
                    acc[mbase + mt][nt] = mma16(fb.get(mt, ks), fa.get(nt, ks), acc[mbase + mt][nt], bf16_t{});
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

    auto last = [&](int t) {
        if (t == steps - 1) sa.last(t), sb.last(t);
    };
    last(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) dma_a(0, i);
    dma_b(0, 0, 0), dma_b(0, 0, 1), dma_b(1, 0, 0), dma_b(1, 0, 1);
    if (steps > 1) {
        last(1);
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
        wait_a();                                                                                 \
        wait_b();                                                                                 \
        multiply(0, (ISSUE_HI) ? 2 : 0, [&](int j) { dma_b(1, t + 1, j); });                      \
        read_b(bo, RG_BHI);                                                                       \
        WAIT_L1;                                                                                  \
        segment_barrier();                                                                        \
        wait_b();                                                                                 \
        if (ISSUE_A) last(t + 2);                                                                 \
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

    const int N = A.rows, M = B.rows;
    char* const stage = smem + wave * OUT_WAVE;
    {
        Residual<64, 64, false> res;
        res.load(epi, g, n0 + wn * 64, m0 + wm * 128, N, M, lane);
        finish_tile<4>([&](int mt, int nt) { return acc[mt][nt]; }, stage, epi, g, split, n0 + wn * 64, m0 + wm * 128, N, M, lane, res);
    }
    Residual<64, 64, false> res;
    res.load(epi, g, n0 + wn * 64, m0 + wm * 128 + 64, N, M, lane);
    finish_tile<4>([&](int mt, int nt) { return acc[4 + mt][nt]; }, stage, epi, g, split, n0 + wn * 64, m0 + wm * 128 + 64, N, M, lane, res);
}

int launch_linear256(const char* what, int mode_a, int mode_b, const Operand& A, const Operand& B, const Epilogue& epi, int64_t K,
                     int64_t KB, const TileGrid& g, hipStream_t s) {
    typedef void (*kern_t)(Operand, Operand, Epilogue, int64_t, int64_t, TileGrid);
    const int which = mode_a == OP_ROWS ? (mode_b == OP_ROWS ? 0 : 1) : 2;
    static const kern_t kerns[3] = {linear256_kernel<OP_ROWS, OP_ROWS>, linear256_kernel<OP_ROWS, OP_COLS>,
                                    linear256_kernel<OP_COLS, OP_COLS>};
    static uint64_t done[3] = {};
    SPHIP_REQUIRE(reserve_lds((const void*)kerns[which], LDS256, done[which]), SPHIP_ELAUNCH, "%s: cannot reserve %d bytes of LDS", what, LDS256);
    const int64_t blocks = (int64_t)g.tilesM * g.tilesN * g.splits;
    hipLaunchKernelGGL(kerns[which], dim3((unsigned)blocks), dim3(512), LDS256, s, A, B, epi, K, KB, g);
    SPHIP_CHECK_LAUNCH(what);
    return SPHIP_OK;
}

}  // namespace sphip
