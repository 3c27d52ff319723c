// The dense product's kernel for small shapes: a 64 x 64 tile of C per workgroup of 4 waves, 128 bytes of K per step (64 bf16,
// 32 fp32), operand tiles by LDS-DMA (images: linear_dma.hpp).
//
// Four times the workgroups of the 128 x 128 kernel, so that a product too small to give every compute unit one of its tiles
// need not split K over workgroups (which costs a round trip of fp32 partial tiles and a second launch). Inside a workgroup
// the waves split K: two halves of the rows of A times two halves of each step's K, 32 x 64 outputs per wave; at the end the
// two waves of a half of the rows exchange 32 of their 64 columns through LDS and each finishes the others (one of them doing
// all 64 took longer: 48 x 768 x 768 with a GELU 8.4 us against 7.2). 4 buffers of 16 KiB, one barrier per step, three steps on their way at any time; two
// workgroups share a compute unit.
#include "linear_dma.hpp"

namespace sphip {

constexpr int T64 = 64, STAGES = 4, STAGE = 16384, IMG_B = 8192;

template <typename T, int MA, int MB, int BYTES>
__global__ __launch_bounds__(256, 2) void linear64_kernel(Operand A, Operand B, Epilogue epi, int64_t K, int64_t KB, TileGrid g) {
    __shared__ __attribute__((aligned(16))) char smem[STAGES * STAGE];
    unsigned split;
    int tm, tn;
    tile_of(g, split, tm, tn);
    const int m0 = tm * T64, n0 = tn * T64;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wn = wave & 1, kh = wave >> 1;
    constexpr int KS = 128 / sizeof(T), PITCH = T64 * sizeof(T);
    const int64_t k0 = (int64_t)split * g.steps_per * KS;
    const int steps = (int)min((int64_t)g.steps_per, (K - k0 + KS - 1) / KS);

    typedef Source<T, MA, T64, BYTES> SA;
    typedef Source<T, MB, T64, BYTES> SB;
    constexpr int LOADS = SA::LOADS + SB::LOADS;   // DMA instructions per wave and step
    SA sa;
    SB sb;
    sa.init(A, n0, k0, K, tid);
    sb.init(B, m0, k0, KB, tid);
    auto fetch = [&](int t, unsigned image) {
        if (t >= steps) return;
        if (t == steps - 1) sa.last(t), sb.last(t);
        char* dst = smem + image + wave * 1024;
        sa.dma(dst, t);
        sb.dma(dst + IMG_B, t);
    };
    const unsigned lds0 = (unsigned)(size_t)(lds_t)smem;
    Frag<T, MA, PITCH, 2> fa;
    Frag<T, MB, PITCH, 4> fb;
    fa.init(lds0, wn * 32, lane, kh);
    fb.init(lds0 + IMG_B, 0, lane, kh);
    acc4_t acc[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i][0] = acc[i][1] = (acc4_t){0.f, 0.f, 0.f, 0.f};

    const int N = A.rows, M = B.rows;
    Residual<32, 32> res;                          // waits in registers until the product is done
    res.load(epi, g, n0 + wn * 32, m0 + kh * 32, N, M, lane);
#pragma unroll
    for (int t = 0; t < STAGES - 1; ++t) fetch(t, t * STAGE);
    unsigned img = 0, freed = (STAGES - 1) * STAGE;            // buffers of step t and of step t - 1
    for (int t = 0; t < steps; ++t) {
        // step t has landed; the at most 2 steps after it that are on their way may still be out
        const int later = steps - 1 - t;
        if (later >= 2) LIN_VMCNT(2 * LOADS);
        else if (later == 1) LIN_VMCNT(LOADS);
        else LIN_VMCNT(0);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        fa.template read<0>(img);
        fb.template read<0>(img);
        fetch(t + STAGES - 1, freed);
        fa.template wait<0, 0>();
        fb.template wait<0, 0>();
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) acc[mt][nt] = mma16(fb.get(mt, 0), fa.get(nt, 0), acc[mt][nt], T{});
        freed = img;
        img = img + STAGE == STAGES * STAGE ? 0 : img + STAGE;
    }
    __syncthreads();                               // the last step has been read: the buffers are free
    acc4_t* const give = reinterpret_cast<acc4_t*>(smem) + wave * 256 + lane;
    const acc4_t* const take = reinterpret_cast<const acc4_t*>(smem) + (wave ^ 2) * 256 + lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) give[i * 64] = kh ? acc[i >> 1][i & 1] : acc[2 + (i >> 1)][i & 1];
    __syncthreads();
    char* const stage = smem + 16384 + wave * 32 * out_row(32);
    const int r16 = lane & 15, q4 = lane >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const acc4_t own = kh ? acc[2 + (i >> 1)][i & 1] : acc[i >> 1][i & 1];
        *reinterpret_cast<acc4_t*>(stage + ((i & 1) * 16 + r16) * out_row(32) + ((i >> 1) * 16 + q4 * 4) * 4) = own + take[i * 64];
    }
    finish_rows(stage, epi, g, split, n0 + wn * 32, m0 + kh * 32, N, M, lane, res);
}

// Splits of the K range: the power of two (or as many as fill the compute units once) with the least time by the step's
// measured 200 ns (bf16; 520 fp32) and, for a split, the joining launch and the partial tiles' round trip (as in linear.hip).
// (Also into more workgroups than there are units, where that leaves them idle for less of the time: fp32 300 x 2048 x 2048 40 us
// whole, 38 in two.)
int linear64_splits(int dtype, int64_t N, int64_t M, int64_t K) {
    const int64_t tiles = cdiv(N, T64) * cdiv(M, T64), steps = cdiv(K, 128 / (int64_t)dtype_size(dtype));
    const int64_t step = dtype == SPHIP_BF16 ? 200 : 520, fill = 256 / tiles < steps / 4 ? 256 / tiles : steps / 4;
    int64_t best = 1, least = steps * step * cdiv(tiles, 256);
    auto consider = [&](int64_t s) {
        const int64_t t = cdiv(steps, s) * step * cdiv(tiles * s, 256) + 3000 + s * N * M / 1000;
        if (t < least) best = s, least = t;
    };
    for (int64_t s = 2; s <= steps / 4 && tiles * s <= 1024; s *= 2) consider(s);
    if (fill > 1) consider(fill);
    return (int)best;
}

int launch_linear64(const char* what, int dtype, int bytes, int mode_a, int mode_b, const Operand& A, const Operand& B,
                    const Epilogue& epi, int64_t K, int64_t KB, const TileGrid& g, hipStream_t s) {
    typedef void (*kern_t)(Operand, Operand, Epilogue, int64_t, int64_t, TileGrid);
    const int64_t blocks = (int64_t)g.tilesM * g.tilesN * g.splits;
    const int which = mode_a == OP_ROWS ? (mode_b == OP_ROWS ? 0 : 1) : 2;
#define LIN_KERNELS(T, BYTES) \
    {linear64_kernel<T, OP_ROWS, OP_ROWS, BYTES>, linear64_kernel<T, OP_ROWS, OP_COLS, BYTES>, linear64_kernel<T, OP_COLS, OP_COLS, BYTES>}
    static const kern_t kerns[3][3] = {LIN_KERNELS(bf16_t, 16), LIN_KERNELS(float, 16), LIN_KERNELS(float, 4)};
#undef LIN_KERNELS
    hipLaunchKernelGGL(kerns[dtype == SPHIP_BF16 ? 0 : bytes == 16 ? 1 : 2][which], dim3((unsigned)blocks), dim3(256), 0, s, A, B, epi, K, KB, g);
    SPHIP_CHECK_LAUNCH(what);
    return SPHIP_OK;
}

}  // namespace sphip
