// The dense product's kernel for mid-size bf16 shapes and for fp32: a 128 x 128 tile of C per workgroup of 4 waves (2 x 2 of
// 64 x 64 outputs), 128 bytes of K per step (64 bf16, 32 fp32), v_mfma_f32_16x16x32_bf16 / v_mfma_f32_16x16x4_f32 (exact
// products, fp32 sums), operand tiles by LDS-DMA (images: linear_dma.hpp).
//
// STAGES buffers of 32 KiB, one barrier per step: at step t a wave waits for its own DMA of step t, passes the barrier
// (everybody's step t has landed, everybody has read step t - 1), sends off the DMA of step t + STAGES - 1 into the buffer
// just freed, reads its fragments and multiplies. With at most one workgroup per compute unit 4 buffers (these shapes are
// short: their time is the latency of the loads), with more 2 buffers, so that two workgroups share a unit and cover each
// other. (32 of K per step with 5 buffers of 16 KiB, two workgroups per unit: 8192 x 2048 x 2048 83 us against 70.)
#include "linear_dma.hpp"

namespace sphip {

constexpr int T128 = 128, IMG_A = 0, IMG_B = 16384, STAGE = 32768;
constexpr int FINISH = 4 * 64 * OUT_ROW;            // the epilogue's staging: more than two stages, twice still within the LDS

template <typename T, int MA, int MB, int STAGES, int BYTES>
__global__ __launch_bounds__(256, STAGES == 2 ? 2 : 1) void linear128_kernel(Operand A, Operand B, Epilogue epi, int64_t K, int64_t KB,
                                                                             TileGrid g) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    unsigned split;
    int tm, tn;
    tile_of(g, split, tm, tn);
    const int m0 = tm * T128, n0 = tn * T128;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    constexpr int KS = 128 / sizeof(T), PITCH = 128 * sizeof(T);
    const int64_t k0 = (int64_t)split * g.steps_per * KS;
    const int steps = (int)min((int64_t)g.steps_per, (K - k0 + KS - 1) / KS);

    typedef Source<T, MA, T128, BYTES> SA;
    typedef Source<T, MB, T128, BYTES> SB;
    constexpr int LOADS = SA::LOADS + SB::LOADS;   // DMA instructions per wave and step
    SA sa;
    SB sb;
    sa.init(A, n0, k0, K, tid);
    sb.init(B, m0, k0, KB, tid);
    auto fetch = [&](int t, unsigned image) {
        if (t >= steps) return;
        if (t == steps - 1) sa.last(t), sb.last(t);
        char* dst = smem + image + wave * 1024;
        sa.dma(dst + IMG_A, t);
        sb.dma(dst + IMG_B, t);
    };
    const unsigned lds0 = (unsigned)(size_t)(lds_t)smem;
    typedef Frag<T, MA, PITCH> FA;
    typedef Frag<T, MB, PITCH> FB;
    FA fa;
    FB fb;
    fa.init(lds0 + IMG_A, wn * 64, lane);
    fb.init(lds0 + IMG_B, wm * 64, lane);
    acc4_t acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = (acc4_t){0.f, 0.f, 0.f, 0.f};

    const int N = A.rows, M = B.rows;
    Residual<64> res;                              // waits in registers until the product is done
    res.load(epi, g, n0 + wn * 64, m0 + wm * 64, N, M, lane);
#pragma unroll
    for (int t = 0; t < STAGES - 1; ++t) fetch(t, t * STAGE);
    unsigned img = 0, freed = (STAGES - 1) * STAGE;            // buffers of step t and of step t - 1
    for (int t = 0; t < steps; ++t) {
        // step t has landed; the (at most STAGES - 2) steps after it that are on their way may still be out
        const int later = min(STAGES - 2, steps - 1 - t);
        if (later == 2) LIN_VMCNT(2 * LOADS);
        else if (later == 1) LIN_VMCNT(LOADS);
        else LIN_VMCNT(0);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        fetch(t + STAGES - 1, freed);
        fa.template read<0>(img);
        fb.template read<0>(img);
        fa.template read<1>(img);
        fb.template read<1>(img);
        constexpr int LATER = FA::READS + FB::READS;     // the counter holds 15 at most
        fa.template wait<0, (LATER > 15 ? 15 : LATER)>();
        fb.template wait<0, (LATER > 15 ? 15 : LATER)>();
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
                acc[mt][nt] = mma16(fb.get(mt, 0), fa.get(nt, 0), acc[mt][nt], T{});
        __builtin_amdgcn_sched_barrier(0);         // these 16 MFMAs run while the other fragments arrive
        fa.template wait<1, 0>();
        fb.template wait<1, 0>();
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int nt = 0; nt < 4; ++nt)
                acc[mt][nt] = mma16(fb.get(mt, 1), fa.get(nt, 1), acc[mt][nt], T{});
        freed = img;
        img = img + STAGE == STAGES * STAGE ? 0 : img + STAGE;
    }
    __syncthreads();                               // the last step has been read: the buffers become the staging area
    finish_tile<4>([&](int mt, int nt) { return acc[mt][nt]; }, smem + wave * 64 * OUT_ROW, epi, g, split, n0 + wn * 64, m0 + wm * 64,
                   N, M, lane, res);
}

// Splits of the K range, towards one workgroup per compute unit, several steps each: a split costs a round trip of the fp32
// partial tiles and the joining launch. bf16: 8 steps (1024^3: 14.9 us, with 2 steps 17.1); a step of fp32 takes 8 times as
// long: 2 steps.
int linear128_splits(int dtype, int64_t N, int64_t M, int64_t K) {
    const int64_t tiles = cdiv(N, T128) * cdiv(M, T128), steps = cdiv(K, 128 / (int64_t)dtype_size(dtype));
    const int64_t least = dtype == SPHIP_BF16 ? 8 : 2;
    int64_t s = 256 / tiles;
    if (s > steps / least) s = steps / least;
    return s < 1 ? 1 : (int)s;
}

int launch_linear128(const char* what, int dtype, int bytes, int mode_a, int mode_b, const Operand& A, const Operand& B,
                     const Epilogue& epi, int64_t K, int64_t KB, const TileGrid& g, hipStream_t s) {
    typedef void (*kern_t)(Operand, Operand, Epilogue, int64_t, int64_t, TileGrid);
    const int64_t blocks = (int64_t)g.tilesM * g.tilesN * g.splits;
    const int which = mode_a == OP_ROWS ? (mode_b == OP_ROWS ? 0 : 1) : 2, deep = blocks <= 256;
    const int type = dtype == SPHIP_BF16 ? 0 : bytes == 16 ? 1 : 2;
#define LIN_KERNELS(T, B)                                                                                       \
    {{linear128_kernel<T, OP_ROWS, OP_ROWS, 2, B>, linear128_kernel<T, OP_ROWS, OP_ROWS, 4, B>},                 \
     {linear128_kernel<T, OP_ROWS, OP_COLS, 2, B>, linear128_kernel<T, OP_ROWS, OP_COLS, 4, B>},                 \
     {linear128_kernel<T, OP_COLS, OP_COLS, 2, B>, linear128_kernel<T, OP_COLS, OP_COLS, 4, B>}}
    static const kern_t kerns[3][3][2] = {LIN_KERNELS(bf16_t, 16), LIN_KERNELS(float, 16), LIN_KERNELS(float, 4)};
#undef LIN_KERNELS
    const int lds = deep ? 4 * STAGE : FINISH;
    static uint64_t done[3][3][2] = {};
    const kern_t fn = kerns[type][which][deep];
    SPHIP_REQUIRE(reserve_lds((const void*)fn, lds, done[type][which][deep]), SPHIP_ELAUNCH, "%s: cannot reserve %d bytes of LDS", what, lds);
    hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3(256), lds, s, A, B, epi, K, KB, g);
    SPHIP_CHECK_LAUNCH(what);
    return SPHIP_OK;
}

}  // namespace sphip
