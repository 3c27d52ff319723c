// Shared by the kernels of the dense product (linear.hip, linear256.hip).
#pragma once
#include "codes8.hpp"
#include "epilogue.hpp"

namespace sphip {

// how element (row, k) of an operand of C[n, m] = sum_k A(n, k) B(m, k) is found
enum { OP_ROWS = 0,      // p[row * ld + k]
       OP_COLS = 1,      // p[k * ld + row]
       OP_COLS_I8 = 2,   // 8-bit codes at p[k * ld + row], scale byte at scales[(k / 32) * ld + row] (checkpoint8.hip)
       OP_COLS_E4M3 = 3 };

struct Operand {
    const void* p;
    const uint8_t* scales;
    int64_t ld;
    int rows;
};

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

// linear256.hip: whether the 256 x 256 kernel takes these operands, how it splits K, and its launch (bf16; the caller joins).
// KB: rows of an OP_COLS B, which may be fewer than K (a multiple of 64 where A is OP_ROWS): B counts as zero from there on.
bool linear256_takes(int mode_a, int mode_b, const Operand& A, const Operand& B, int64_t K);
int linear256_splits(int64_t N, int64_t M, int64_t K);
int launch_linear256(const char* what, int mode_a, int mode_b, const Operand& A, const Operand& B, const Epilogue& epi, int64_t K,
                     int64_t KB, const TileGrid& g, hipStream_t s);

}  // namespace sphip
