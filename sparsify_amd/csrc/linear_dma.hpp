// LDS-DMA staging and fragment reads shared by the dense product's kernels (linear64.hip, linear128.hip: bf16, fp32;
// linear256.hip: bf16).
//
// An operand is either contiguous in K (OP_ROWS: image [row][8 chunks of 8 k], chunk XOR (row >> 1) & 7, ds_read_b128) or
// contiguous in its rows (OP_COLS: the gradient products). The latter is not transposed in memory: its image is [k][chunks
// of 8 rows] as it comes, and ds_read_b64_tr_b16 hands every lane 4 consecutive k of its row (of 16 lanes, lane i names
// k = i / 4 and rows 4 (i % 4) .. + 3 and receives row i). Chunk XOR 2 ((k & 3) + 4 ((k >> 3) & 1)) spreads the 4 k of one
// read, and the 8 apart ones of the neighbouring 16 lanes, over 8 different 32-byte slots: no bank conflicts (cols_swizzle).
// LDS-DMA writes linearly, so both swizzles are applied to the per-lane source address; rows and K past the end read as
// zeros by the buffer descriptors' range check (K past the end of an OP_ROWS operand is the next row's memory: last()).
#pragma once
#include "linear.hpp"

namespace sphip {

constexpr int K64 = 64;                            // bf16 K per step: 128 bytes (32 fp32)
constexpr unsigned PAST_END = 1u << 31;            // offset bit that lies behind every descriptor (MAX_LD)

#define LIN_VMCNT(n) asm volatile("s_waitcnt vmcnt(%0)" ::"i"((n) < 63 ? (n) : 63) : "memory")     // (6 bits)

// Chunk swizzle of an OP_COLS image with PITCH bytes per k row, element size ES (see above; with 128-byte rows the low bit of
// k already tells the two halves of the banks apart, and fp32 reads single dwords: there the four 16-lane groups, 4 k rows
// apart, go to different 64-byte quarters).
template <int ES, int PITCH> __device__ __forceinline__ int cols_swizzle(int k) {
    if (ES == 4) return 4 * ((k >> 2) & 3);
    if (PITCH == 128) return 2 * (((k >> 1) & 1) + 2 * ((k >> 3) & 1));
    return 2 * ((k & 3) + 4 * ((k >> 3) & 1));
}

// TILES 16-row fragments of a 128-byte K step, the reads of one half (32 bf16 k, 16 fp32 k) at a time: read<0>(), read<1>(),
// wait<H, COUNT>() once at most COUNT later LDS operations are outstanding. Issued from inline asm (the compiler would drain
// the DMA queue before each LDS read it sees); wait() passes every destination register of the half through an asm statement
// behind its s_waitcnt, so that nothing reads one before. init(): the wave's rows start at row0 of the image, half 0 is `h0`.
template <typename T, int MODE, int PITCH, int TILES = 4> struct Frag;
template <typename T, int PITCH, int TILES> struct Frag<T, OP_ROWS, PITCH, TILES> {
    static constexpr int READS = TILES;                // LDS operations per half
    w4_t v[TILES][2];
    unsigned a[2];                                     // the lane's address per half; tiles are 16 rows = 2048 bytes apart
    __device__ __forceinline__ void init(unsigned lds0, int row0, int lane, int h0 = 0) {
        const int r16 = lane & 15, q4 = lane >> 4;
#pragma unroll
        for (int h = 0; h < 2; ++h) a[h] = lds0 + (row0 + r16) * 128 + (((4 * (h ^ h0) + q4) ^ ((r16 >> 1) & 7)) << 4);
    }
    template <int H> __device__ __forceinline__ void read(unsigned image) {
        const unsigned at = a[H] + image;
#define LIN_DSR(i) \
    if constexpr (i < TILES) asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(v[i][H]) : "v"(at), "i"((i) * 2048))
        LIN_DSR(0); LIN_DSR(1); LIN_DSR(2); LIN_DSR(3);
#undef LIN_DSR
    }
    template <int H, int COUNT> __device__ __forceinline__ void wait() {
        asm volatile("s_waitcnt lgkmcnt(%0)" ::"i"(COUNT));
#pragma unroll
        for (int i = 0; i < TILES; ++i) asm volatile("" : "+v"(v[i][H]));
    }
    __device__ __forceinline__ w4_t get(int i, int h) const { return v[i][h]; }
};
template <int PITCH, int TILES> struct Frag<bf16_t, OP_COLS, PITCH, TILES> {
    static constexpr int READS = 2 * TILES;
    w2_t v[TILES][2][2];                               // [tile][half][4-k quarter]
    unsigned a[TILES];                                 // the lane's address per tile
    __device__ __forceinline__ void init(unsigned lds0, int row0, int lane, int h0 = 0) {
        const int r16 = lane & 15, q4 = lane >> 4, k = 8 * q4 + (r16 >> 2);
#pragma unroll
        for (int i = 0; i < TILES; ++i)
            a[i] = lds0 + (k + 32 * h0) * PITCH + (((row0 / 8 + 2 * i + ((r16 & 3) >> 1)) ^ cols_swizzle<2, PITCH>(k)) << 4) + (r16 & 1) * 8;
    }
    template <int H> __device__ __forceinline__ void read(unsigned image) {
#define LIN_DSR(i, q)                                                                                            \
    if constexpr (i < TILES)                                                                                     \
        asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v[i][H][q]) : "v"(a[i] + image), "i"(H * 32 * PITCH + (q) * 4 * PITCH))
        LIN_DSR(0, 0); LIN_DSR(0, 1); LIN_DSR(1, 0); LIN_DSR(1, 1);
        LIN_DSR(2, 0); LIN_DSR(2, 1); LIN_DSR(3, 0); LIN_DSR(3, 1);
#undef LIN_DSR
    }
    template <int H, int COUNT> __device__ __forceinline__ void wait() {
        asm volatile("s_waitcnt lgkmcnt(%0)" ::"i"(COUNT));
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            asm volatile("" : "+v"(v[i][H][0]));
            asm volatile("" : "+v"(v[i][H][1]));
        }
    }
    __device__ __forceinline__ w4_t get(int i, int h) const { return __builtin_shufflevector(v[i][h][0], v[i][h][1], 0, 1, 2, 3); }
};
// fp32 needs no transposing read: a lane's 4 k (4 (4 h + q4) + j, as in the OP_ROWS image) are 4 dwords of its column
template <int PITCH, int TILES> struct Frag<float, OP_COLS, PITCH, TILES> {
    static constexpr int READS = 4 * TILES;
    unsigned v[TILES][2][4];
    unsigned a[TILES];
    __device__ __forceinline__ void init(unsigned lds0, int row0, int lane, int h0 = 0) {
        const int r16 = lane & 15, q4 = lane >> 4;
#pragma unroll
        for (int i = 0; i < TILES; ++i)
            a[i] = lds0 + (4 * q4 + 16 * h0) * PITCH + (((row0 / 4 + 4 * i + (r16 >> 2)) ^ cols_swizzle<4, PITCH>(4 * q4)) << 4) + (r16 & 3) * 4;
    }
    template <int H> __device__ __forceinline__ void read(unsigned image) {
#define LIN_DSR(i, j)        \
    if constexpr (i < TILES) \
        asm volatile("ds_read_b32 %0, %1 offset:%2" : "=v"(v[i][H][j]) : "v"(a[i] + image), "i"(H * 16 * PITCH + (j) * PITCH))
        LIN_DSR(0, 0); LIN_DSR(0, 1); LIN_DSR(0, 2); LIN_DSR(0, 3); LIN_DSR(1, 0); LIN_DSR(1, 1); LIN_DSR(1, 2); LIN_DSR(1, 3);
        LIN_DSR(2, 0); LIN_DSR(2, 1); LIN_DSR(2, 2); LIN_DSR(2, 3); LIN_DSR(3, 0); LIN_DSR(3, 1); LIN_DSR(3, 2); LIN_DSR(3, 3);
#undef LIN_DSR
    }
    template <int H, int COUNT> __device__ __forceinline__ void wait() {
        asm volatile("s_waitcnt lgkmcnt(%0)" ::"i"(COUNT));
#pragma unroll
        for (int i = 0; i < TILES; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(v[i][H][j]));
    }
    __device__ __forceinline__ w4_t get(int i, int h) const { return (w4_t){v[i][h][0], v[i][h][1], v[i][h][2], v[i][h][3]}; }
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
template <int NT, typename Acc, bool BIAS>
__device__ __forceinline__ void finish_tile(Acc acc, char* stage, const Epilogue& epi, const TileGrid& g, unsigned split, int n0,
                                            int m0, int N, int M, int lane, const Residual<NT * 16, 64, BIAS>& res) {
    const int r16 = lane & 15, q4 = lane >> 4;
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            *reinterpret_cast<acc4_t*>(stage + (nt * 16 + r16) * OUT_ROW + (mt * 16 + q4 * 4) * 4) = acc(mt, nt);
    finish_rows(stage, epi, g, split, n0, m0, N, M, lane, res);
}

// One operand of a kernel of 256 threads, TILE rows: descriptor, the lane's source offsets, the DMA of one 128-byte K step
// (PIECES times 4 KiB per workgroup, an instruction BYTES per lane). BYTES 16: rows from multiples of 16 bytes, K whole such
// pieces where it is contiguous; BYTES 4: fp32 at any address (four times the instructions: 2048 x 1025 x 1024 44 us; copied
// first, then by 16 bytes, 50; 98 x 5502 x 7155 118 against 173).
template <typename T, int MODE, int TILE, int BYTES> struct Source {
    static constexpr unsigned ES = sizeof(T), KS = 128 / ES;
    static constexpr int PIECES = TILE / 32, PITCH = TILE * ES, J = 16 / BYTES, ALT = MODE == OP_ROWS ? 1 : 2;
    static constexpr int LOADS = PIECES * J;                    // instructions per wave and step
    const T* base;                         // of the tile and the split, uniform
    unsigned ldb, edge;                    // bytes: row stride; OP_ROWS: of the descriptor, OP_COLS: of its last k row
    unsigned voff[ALT][J], piece;          // bytes: lane offset of even and odd pieces, between pieces
    int left[J];                           // OP_ROWS: K from the lane's on in units of BYTES; OP_COLS: k rows
    __device__ __forceinline__ void init(const Operand& o, int row0, int64_t k0, int64_t K, int tid) {
        ldb = (unsigned)o.ld * ES;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            // the 16-byte slot of the image the lane writes (a part of) with load j of a piece
            const int u = J == 1 ? tid : (tid & ~63) + j * 16 + ((tid & 63) >> 2), sub = J == 1 ? 0 : (tid & 3) * 4;
            if (MODE == OP_ROWS) {
                const int hr = u >> 3, ch = (u & 7) ^ ((hr >> 1) & 7);
                voff[0][j] = (unsigned)hr * ldb + (unsigned)(ch * 16 + sub);
                left[j] = (int)((K - k0) * ES / BYTES) - (ch * 16 + sub) / BYTES;
            } else {
                constexpr int CH = PITCH / 16, KP = 256 / CH;   // 16-byte chunks of a k row, k rows of a piece
                const int kr = u / CH, c = u % CH;
#pragma unroll
                for (int i = 0; i < ALT; ++i) voff[i][j] = (unsigned)kr * ldb + (unsigned)((c ^ cols_swizzle<ES, PITCH>(kr + KP * i)) * 16 + sub);
                piece = KP * ldb;
                left[j] = (int)(K - k0);
            }
        }
        if (MODE == OP_ROWS) {
            base = (const T*)o.p + (int64_t)row0 * o.ld + k0;
            edge = (unsigned)(min(TILE, o.rows - row0) - 1) * ldb + (unsigned)(K - k0) * ES;
            piece = 32u * ldb;
        } else {
            base = (const T*)o.p + k0 * o.ld + row0;
            // rounded up to what a lane loads: a dword that crosses the end reads as zero, with it the last of an odd number of
            // rows (k rows are 16-byte aligned then, so the piece is the one that holds the last element)
            edge = ((unsigned)(o.rows - row0) * ES + (BYTES - 1u)) / BYTES * BYTES;
        }
    }
    // The descriptor of K step t. OP_COLS: from the step's first k row, so that its offsets do not grow with K (many tokens).
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t step(int t) const {
        if (MODE == OP_ROWS) return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)edge, 0x00020000);
        const unsigned rows = (unsigned)min((int)KS, left[0] - t * (int)KS);
        return __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)base + (uint64_t)((unsigned)t * KS) * ldb), 0,
                                                 (int)((rows - 1) * ldb + edge), 0x00020000);
    }
    // before the DMA of the last step: an OP_ROWS lane whose piece lies behind K names an offset behind the descriptor
    __device__ __forceinline__ void last(int t) {
        if (MODE == OP_ROWS)
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (128 / BYTES * t >= left[j]) voff[0][j] |= PAST_END;
    }
    __device__ __forceinline__ void dma(char* lds, int t) const {
        const __amdgpu_buffer_rsrc_t rsrc = step(t);
        const unsigned so = MODE == OP_ROWS ? (unsigned)t * 128u : 0u;
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
            for (int j = 0; j < J; ++j) {     // (the whole offset in the register the range check looks at)
                const lds_t to = (lds_t)(lds + 4096 * i + 1024 / J * j);
                const unsigned from = voff[i & (ALT - 1)][j] + (unsigned)i * piece + so;
                if constexpr (BYTES == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, to, 16, from, 0, 0, 0);
                else __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, to, 4, from, 0, 0, 0);
            }
    }
};

}  // namespace sphip
