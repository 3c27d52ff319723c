// LDS-DMA staging and fragment reads shared by the dense product's kernels (linear256.hip: bf16, linear128.hip: bf16, fp32).
//
// An operand is either contiguous in K (OP_ROWS: image [row][8 chunks of 8 k], chunk XOR (row >> 1) & 7, ds_read_b128) or
// contiguous in its rows (OP_COLS: the gradient products). The latter is not transposed in memory: its image is [k][chunks
// of 8 rows] as it comes, and ds_read_b64_tr_b16 hands every lane 4 consecutive k of its row (of 16 lanes, lane i names
// k = i / 4 and rows 4 (i % 4) .. + 3 and receives row i). Chunk XOR 2 ((k & 3) + 4 ((k >> 3) & 1)) spreads the 4 k of one
// read, and the 8 apart ones of the neighbouring 16 lanes, over 8 different 32-byte slots: no bank conflicts.
// LDS-DMA writes linearly, so both swizzles are applied to the per-lane source address; rows and K past the end read as
// zeros by the buffer descriptors' range check (K past the end of an OP_ROWS operand does not, hence K % 64 == 0 there).
#pragma once
#include "linear.hpp"

namespace sphip {

constexpr int K64 = 64;                            // bf16 K per step: 128 bytes (32 fp32)

#define LIN_VMCNT(n) asm volatile("s_waitcnt vmcnt(" #n ")" ::: "memory")

// Four 16-row fragments of 64 k, the reads of one 32-k step at a time: read<0>(), read<1>(), wait<KS, COUNT>() once at most
// COUNT later LDS operations are outstanding. Issued from inline asm (the compiler would drain the DMA queue before each
// LDS read it sees); the wait names the step's destination registers, so that nothing reads them before.
template <typename T, int MODE, int PITCH> struct Frag;
template <typename T, int PITCH> struct Frag<T, OP_ROWS, PITCH> {
    static constexpr int READS = 4;                    // LDS operations per 32-k step
    w4_t v[4][2];
    unsigned a[2];                                     // the lane's address per 32-k step; tiles are 16 rows = 2048 bytes apart
    // the wave's 64 rows start at row0 of the image
    __device__ __forceinline__ void init(unsigned lds0, int row0, int lane) {
        const int r16 = lane & 15, q4 = lane >> 4;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) a[ks] = lds0 + (row0 + r16) * 128 + (((4 * ks + q4) ^ ((r16 >> 1) & 7)) << 4);
    }
    template <int KS> __device__ __forceinline__ void read(unsigned image) {
        const unsigned at = a[KS] + image;
#define LIN_DSR(i) asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v[i][KS]) : "v"(at), "i"((i) * 2048))
        LIN_DSR(0); LIN_DSR(1); LIN_DSR(2); LIN_DSR(3);
#undef LIN_DSR
    }
    template <int KS, int COUNT> __device__ __forceinline__ void wait() {
        asm volatile("s_waitcnt lgkmcnt(%4)" : "+v"(v[0][KS]), "+v"(v[1][KS]), "+v"(v[2][KS]), "+v"(v[3][KS]) : "i"(COUNT));
    }
    __device__ __forceinline__ w4_t get(int i, int ks) const { return v[i][ks]; }
};
template <int PITCH> struct Frag<bf16_t, OP_COLS, PITCH> {      // PITCH bytes per k row of the image
    static constexpr int READS = 8;
    w2_t v[4][2][2];                                   // [tile][32-k step][4-k half]
    unsigned a[4];                                     // the lane's address per tile
    __device__ __forceinline__ void init(unsigned lds0, int row0, int lane) {
        const int r16 = lane & 15, q4 = lane >> 4;
        const int k = 8 * q4 + (r16 >> 2), f = (k & 3) + 4 * ((k >> 3) & 1);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            a[i] = lds0 + k * PITCH + (((row0 / 8 + 2 * i + ((r16 & 3) >> 1)) ^ (2 * f)) << 4) + (r16 & 1) * 8;
    }
    template <int KS> __device__ __forceinline__ void read(unsigned image) {
#define LIN_DSR(i, h)                                                                                            \
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2"                                                           \
                 : "=v"(v[i][KS][h])                                                                             \
                 : "v"(a[i] + image), "i"(KS * 32 * PITCH + (h) * 4 * PITCH))
        LIN_DSR(0, 0); LIN_DSR(0, 1); LIN_DSR(1, 0); LIN_DSR(1, 1);
        LIN_DSR(2, 0); LIN_DSR(2, 1); LIN_DSR(3, 0); LIN_DSR(3, 1);
#undef LIN_DSR
    }
    template <int KS, int COUNT> __device__ __forceinline__ void wait() {
        asm volatile("s_waitcnt lgkmcnt(%8)"
                     : "+v"(v[0][KS][0]), "+v"(v[0][KS][1]), "+v"(v[1][KS][0]), "+v"(v[1][KS][1]), "+v"(v[2][KS][0]),
                       "+v"(v[2][KS][1]), "+v"(v[3][KS][0]), "+v"(v[3][KS][1])
                     : "i"(COUNT));
    }
    __device__ __forceinline__ w4_t get(int i, int ks) const { return __builtin_shufflevector(v[i][ks][0], v[i][ks][1], 0, 1, 2, 3); }
};
// fp32 needs no transposing read: a lane's 4 k (4 (4 ks + q4) + j, as in the OP_ROWS image) are 4 dwords of its column.
// Chunk XOR 4 ((k >> 2) & 3): the four 16-lane groups, 4 k rows apart, read different 64-byte quarters of the banks.
template <int PITCH> struct Frag<float, OP_COLS, PITCH> {
    static constexpr int READS = 16;
    unsigned v[4][2][4];
    unsigned a[4];
    __device__ __forceinline__ void init(unsigned lds0, int row0, int lane) {
        const int r16 = lane & 15, q4 = lane >> 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = lds0 + 4 * q4 * PITCH + (((row0 / 4 + 4 * i + (r16 >> 2)) ^ (4 * q4)) << 4) + (r16 & 3) * 4;
    }
    template <int KS> __device__ __forceinline__ void read(unsigned image) {
#define LIN_DSR(i, j) \
    asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(v[i][KS][j]) : "v"(a[i] + image), "i"(KS * 16 * PITCH + (j) * PITCH))
        LIN_DSR(0, 0); LIN_DSR(0, 1); LIN_DSR(0, 2); LIN_DSR(0, 3); LIN_DSR(1, 0); LIN_DSR(1, 1); LIN_DSR(1, 2); LIN_DSR(1, 3);
        LIN_DSR(2, 0); LIN_DSR(2, 1); LIN_DSR(2, 2); LIN_DSR(2, 3); LIN_DSR(3, 0); LIN_DSR(3, 1); LIN_DSR(3, 2); LIN_DSR(3, 3);
#undef LIN_DSR
    }
    template <int KS, int COUNT> __device__ __forceinline__ void wait() {
        asm volatile("s_waitcnt lgkmcnt(%16)"
                     : "+v"(v[0][KS][0]), "+v"(v[0][KS][1]), "+v"(v[0][KS][2]), "+v"(v[0][KS][3]), "+v"(v[1][KS][0]), "+v"(v[1][KS][1]),
                       "+v"(v[1][KS][2]), "+v"(v[1][KS][3]), "+v"(v[2][KS][0]), "+v"(v[2][KS][1]), "+v"(v[2][KS][2]),
                       "+v"(v[2][KS][3]), "+v"(v[3][KS][0]), "+v"(v[3][KS][1]), "+v"(v[3][KS][2]), "+v"(v[3][KS][3])
                     : "i"(COUNT));
    }
    __device__ __forceinline__ w4_t get(int i, int ks) const { return (w4_t){v[i][ks][0], v[i][ks][1], v[i][ks][2], v[i][ks][3]}; }
};

// c += a b^T over 16 bytes of K per lane (32 bf16 k, or 16 fp32 k in four 4-wide MFMAs: element j of every lane each time)
__device__ __forceinline__ acc4_t mma16(const w4_t& a, const w4_t& b, acc4_t c, bf16_t) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8_t, a), __builtin_bit_cast(b16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ acc4_t mma16(const w4_t& a, const w4_t& b, acc4_t c, float) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[j]), __uint_as_float(b[j]), c, 0, 0, 0);
    return c;
}

// The 16x16 accumulators acc(mt, nt) of a wave (4 consecutive m of one n per lane), 16 NT rows of n, through its LDS area.
template <int NT, typename Acc>
__device__ __forceinline__ void finish_tile(Acc acc, char* stage, const Epilogue& epi, const TileGrid& g, unsigned split, int n0,
                                            int m0, int N, int M, int lane, const Residual<NT * 16>& res) {
    const int r16 = lane & 15, q4 = lane >> 4;
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            *reinterpret_cast<acc4_t*>(stage + (nt * 16 + r16) * OUT_ROW + (mt * 16 + q4 * 4) * 4) = acc(mt, nt);
    finish_rows<NT * 16>(stage, epi, g, split, n0, m0, N, M, lane, res);
}

// whether LDS-DMA can fetch an operand of es-byte elements: 16-byte aligned rows, 32-bit byte offsets inside a tile's
// descriptor, whole 128-byte steps of K where K is the contiguous index
static inline bool dma_ok(int mode, const Operand& o, int64_t K, int tile, int es) {
    if (((uintptr_t)o.p & 15) != 0 || o.ld * es % 16 != 0) return false;
    if (mode == OP_ROWS) return K * es % 128 == 0 && (o.ld * tile + K) * es < (1ll << 31);
    return mode == OP_COLS && (K + 128 / es) * o.ld * es < (1ll << 31);
}

}  // namespace sphip
