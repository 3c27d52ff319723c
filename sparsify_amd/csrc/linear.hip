// A dense product with bias, activation and residual in its epilogue, and its gradients:
//     y = act(x W^T + b) + r                                            (sphip_linear)
//     dz = g act'(z), db = sum_n dz, dx = dz W, dW = dz^T x             (sphip_linear_backward)
// x and z as they are or as 8-bit checkpoints (checkpoint8.hip).
// The skip connection of a transcoder (sparsify/sparse_coder.py:219-222) is the first user, in coders that keep their input in
// 8 bits.
//
// All three products are C[n, m] = sum_k A(n, k) B(m, k); what differs is which index of an operand is contiguous in memory.
// linear64.hip, linear128.hip and linear256.hip are one tiling each, linear_few.hip is for few rows; this file chooses, copies
// what LDS-DMA cannot fetch as it is (linear_pack_kernel), restores 8-bit codes, computes dz and db, and joins the fp32
// partial tiles of a K range split over workgroups, in a fixed order.
#include "linear.hpp"
#include <stdlib.h>

namespace sphip {

// Sum of the splits' partial tiles, then the epilogue. One thread per 4 outputs, the splits in order; with many splits of a
// small product 8 threads share an output, each taking every eighth split (LANES = 8), their sums added in order.
template <int LANES>
__global__ __launch_bounds__(256) void linear_join_kernel(const float* __restrict__ part, Epilogue epi, int64_t N, int M,
                                                          int splits) {
    constexpr int OUTS = 256 / LANES;
    __shared__ float4 red[LANES][OUTS];
    const int quads = (M + 3) >> 2, lane = threadIdx.x / OUTS, o = threadIdx.x % OUTS;
    const int64_t i = (int64_t)blockIdx.x * OUTS + o, total = N * quads;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (i < total) {
#pragma unroll 4
        for (int s = lane; s < splits; s += LANES) {
            const float4 t = load4(part + (s * total + i) * 4);
            v[0] += t.x, v[1] += t.y, v[2] += t.z, v[3] += t.w;
        }
    }
    if (LANES > 1) {
        red[lane][o] = make_float4(v[0], v[1], v[2], v[3]);
        __syncthreads();
        if (lane != 0) return;
#pragma unroll
        for (int l = 1; l < LANES; ++l) {
            const float4 t = red[l][o];
            v[0] += t.x, v[1] += t.y, v[2] += t.z, v[3] += t.w;
        }
    }
    if (i < total) epilogue4(epi, i / quads, (int)(i % quads) * 4, M, v);
}

static size_t part_bytes(int64_t N, int64_t M, int splits) {
    return splits > 1 ? (size_t)splits * N * ((M + 3) / 4 * 4) * 4 : 0;
}
// SPHIP_LINEAR=64|128|256|few forces a kernel (tests, A/B runs); read once per entry point
static thread_local char g_forced = 0;
static void read_forced() {
    const char* e = getenv("SPHIP_LINEAR");
    g_forced = e ? e[0] : 0;
}

// which kernel a product of these sizes goes to
enum { BY_64 = 1, BY_128 = 2, BY_256 = 3 };
static int splits_of(int dtype, int by, int64_t N, int64_t M, int64_t K) {
    return by == BY_256 ? 1 : by == BY_128 ? linear128_splits(dtype, N, M, K) : linear64_splits(dtype, N, M, K);
}
// Time of a product with 64 x 64 or 128 x 128 tiles in ns, without what both take: K steps one after the other, a step of one
// workgroup `step` (measured: 64 x 64 200 bf16, 520 fp32; 128 x 128 570 and 2100 alone on its compute unit, 400 and 1950 where
// two share one), 1.2 us more of filling and finishing for the larger tile, and for a split K range 3 us of joining launch
// and a round trip of the partial tiles at 8 TB/s (they stay in the Infinity Cache: 100 x 7152 x 5504 31 us whole, 25 split).
static int64_t product_ns(int dtype, int by, int64_t N, int64_t M, int64_t K) {
    const int64_t tile = by == BY_64 ? 64 : 128, splits = splits_of(dtype, by, N, M, K);
    const int64_t groups = cdiv(N, tile) * cdiv(M, tile) * splits, steps = cdiv(cdiv(K, 128 / (int64_t)dtype_size(dtype)), splits);
    const bool bf = dtype == SPHIP_BF16;
    const int64_t step = by == BY_64 ? (bf ? 200 : 520) : groups <= 256 ? (bf ? 570 : 2100) : (bf ? 400 : 1950);
    return steps * step * cdiv(groups, 256) + (by == BY_64 ? 0 : 1200) + (splits > 1 ? 3000 + splits * N * M / 1000 : 0);
}
static int kernel_for(int dtype, int64_t N, int64_t M, int64_t K) {
    if (g_forced == '6') return BY_64;
    if (g_forced == '1' || g_forced == '2') return g_forced == '2' && dtype == SPHIP_BF16 ? BY_256 : BY_128;
    // The 256 x 256 kernel where its tiles fill most of the 256 compute units once: 16384 x 1024 x 4096 takes 117 us against
    // 136 with 128 x 128 tiles, 8192 x 2048 x 2048 53 against 62; with fewer the smaller tiles win (2048^3 24 against 37).
    if (dtype == SPHIP_BF16 && cdiv(N, 256) * cdiv(M, 256) >= 160) return BY_256;
    // 64 against 128: 1024^3 7.1 us / 14.9, 2048 x 512 x 512 in fp32 13 / 24, 1003 x 769 x 2050 with bias, SiLU and residual
    // 22.5 / 25.1, but 2048^3 27 / 24 and 16384 tokens' gradient of a 768 x 768 weight 56 / 32
    return product_ns(dtype, BY_64, N, M, K) <= product_ns(dtype, BY_128, N, M, K) ? BY_64 : BY_128;
}

// what a product needs for its partial tiles
static size_t split_bytes(int dtype, int64_t N, int64_t M, int64_t K) {
    const int64_t Kp = cdiv(K, 64) * 64;
    return part_bytes(N, M, splits_of(dtype, kernel_for(dtype, N, M, Kp), N, M, Kp));
}

template <typename T, int MODE_A, int MODE_B>
static int launch_product(const char* what, const Operand& A, const Operand& B, const Epilogue& epi, int64_t K, int64_t KB,
                          void* ws, size_t ws_bytes, hipStream_t s) {
    const int64_t N = A.rows, M = B.rows;
    constexpr int dtype = sizeof(T) == 2 ? SPHIP_BF16 : SPHIP_F32;
    const int by = kernel_for(dtype, N, M, cdiv(K, 64) * 64);
    const int tile = by == BY_256 ? 256 : by == BY_64 ? 64 : 128;
    const int64_t steps = cdiv(K, 128 / (int64_t)sizeof(T));
    TileGrid g;
    g.tilesM = (int)cdiv(M, tile), g.tilesN = (int)cdiv(N, tile);
    const int want = splits_of(dtype, by, N, M, cdiv(K, 64) * 64);
    g.steps_per = (int)cdiv(steps, want);
    g.splits = (int)cdiv(steps, g.steps_per);
    g.part = (float*)ws;
    if (g.splits > 1) {
        const size_t need = part_bytes(N, M, g.splits);
        SPHIP_REQUIRE(ws != nullptr && ws_bytes >= need && ((uintptr_t)ws & 15) == 0, SPHIP_EWORKSPACE,
                      "%s: workspace of %zu bytes, needs %zu, 16-byte aligned", what, ws_bytes, need);
    }
    const int64_t nblocks = (int64_t)g.tilesM * g.tilesN * g.splits, threads = N * ((M + 3) / 4);
    SPHIP_REQUIRE(nblocks < MAX_GROUPS && (g.splits == 1 || cdiv(threads, 256) < MAX_GROUPS), SPHIP_EUNSUPPORTED,
                  "%s: grid too large", what);
    const int bytes = aligned16(A.p, A.ld, sizeof(T)) && aligned16(B.p, B.ld, sizeof(T)) && (MODE_A == OP_COLS || K * (int64_t)sizeof(T) % 16 == 0) ? 16 : 4;
    const int st = by == BY_256 ? launch_linear256(what, MODE_A, MODE_B, A, B, epi, K, KB, g, s)
                 : by == BY_128 ? launch_linear128(what, dtype, bytes, MODE_A, MODE_B, A, B, epi, K, KB, g, s)
                                : launch_linear64(what, dtype, bytes, MODE_A, MODE_B, A, B, epi, K, KB, g, s);
    if (st != SPHIP_OK) return st;
    if (g.splits > 1) {
        if (g.splits > 8 && threads < (1 << 17))
            hipLaunchKernelGGL(linear_join_kernel<8>, dim3((unsigned)cdiv(threads, 32)), dim3(256), 0, s, g.part, epi, N, (int)M, g.splits);
        else
            hipLaunchKernelGGL(linear_join_kernel<1>, dim3((unsigned)cdiv(threads, 256)), dim3(256), 0, s, g.part, epi, N, (int)M, g.splits);
        SPHIP_CHECK_LAUNCH(what);
    }
    return SPHIP_OK;
}

// Rows copied to a stride that is a multiple of 64 elements, zeros behind them: for operands that LDS-DMA cannot fetch as they
// are (fetchable(); bf16 products of K from D or M also need rows that are whole 16-byte pieces). Up to three matrices in one
// launch.
struct PackArgs {
    const void* src[3];
    void* dst[3];
    int64_t ld[3], rows[3];
    int cols[3], pieces[3], log[3];        // 16-byte pieces per row; a row is taken by 2^log threads of a workgroup
    unsigned first[3];                     // the first workgroup of each (of none: behind the last)
};
template <typename T> __global__ __launch_bounds__(256) void linear_pack_kernel(PackArgs a) {
    constexpr int E = 16 / sizeof(T);
    const int w = (int)(blockIdx.x >= a.first[1]) + (int)(blockIdx.x >= a.first[2]);
    const int64_t row = ((int64_t)(blockIdx.x - a.first[w]) << (8 - a.log[w])) + (threadIdx.x >> a.log[w]);
    if (row >= a.rows[w]) return;
    const int cols = a.cols[w], pieces = a.pieces[w];
    const T* src = (const T*)a.src[w] + row * a.ld[w];
    uint4* dst = (uint4*)a.dst[w] + row * pieces;
#pragma unroll 2
    for (int i = (int)threadIdx.x & ((1 << a.log[w]) - 1); i < pieces; i += 1 << a.log[w]) {
        const int c = i * E, miss = max(c + E - cols, 0);
        unsigned v[4] = {0, 0, 0, 0};
        if (c < cols) {
            if (cols >= E) {
                __builtin_memcpy(v, src + c - miss, 16);
                if (miss > 0) drop_front(v, miss * (int)sizeof(T));
            } else {
                load_short(src, cols, v);
            }
        }
        dst[i] = make_uint4(v[0], v[1], v[2], v[3]);
    }
}
static int64_t packed_ld(int64_t cols) { return cdiv(cols, 64) * 64; }
static int64_t whole_pieces(int64_t cols) { return cdiv(cols, 8) * 8; }
struct Packing {
    PackArgs a = {};
    int count = 0, dtype;
    explicit Packing(int dt) : dtype(dt) {}
    void add(Operand& o, int64_t rows, int64_t cols, void* dst) {
        const int64_t ld = packed_ld(cols);
        a.src[count] = o.p, a.dst[count] = dst, a.ld[count] = o.ld, a.rows[count] = rows, a.cols[count] = (int)cols;
        a.pieces[count] = (int)(ld * (int64_t)dtype_size(dtype) / 16);
        while (a.log[count] < 8 && (1 << a.log[count]) < a.pieces[count]) ++a.log[count];
        ++count;
        o.p = dst, o.ld = ld;
    }
    int launch(const char* what, hipStream_t s) {
        if (count == 0) return SPHIP_OK;
        int64_t blocks = 0;
        for (int i = 0; i < 3; ++i) {
            a.first[i] = (unsigned)blocks;
            if (i < count) blocks += cdiv(a.rows[i], 256 >> a.log[i]);
            SPHIP_REQUIRE(blocks < MAX_GROUPS, SPHIP_EUNSUPPORTED, "%s: grid too large", what);
        }
        if (dtype == SPHIP_BF16) hipLaunchKernelGGL(linear_pack_kernel<bf16_t>, dim3((unsigned)blocks), dim3(256), 0, s, a);
        else hipLaunchKernelGGL(linear_pack_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, s, a);
        SPHIP_CHECK_LAUNCH(what);
        return SPHIP_OK;
    }
};
// whether rows of so many elements end inside a 16-byte piece that LDS-DMA would fetch whole
static bool unaligned(int dtype, int64_t cols) { return dtype == SPHIP_BF16 && cols % 8 != 0; }

// ---- dz = g act'(z) and its column sums. A workgroup takes 32 rows (the group one scale of an 8-bit z covers) of 32 x 16
// bytes of columns: 32 lanes side by side, 8 rows at a time, every thread 4 rows whose loads are all in flight; the 8 row
// sums of a column meet in LDS and go to part[row group][M], added up in order by the second kernel.
// dz leaves in the products' type: a bf16 MFMA takes no more, and the remainder in a second bf16 product would double the
// time. Rounding it once adds to dx and dW what their own rounding to bf16 does (16384 x 4096 x 4096: 0.0023 from the 64-bit
// gradients against 0.0017 with dz in fp32, root mean square). db sums dz before it is rounded.
struct PreactArgs {
    const void* g;
    const void* z;                 // values or codes, row stride ldz
    const uint8_t* scales;
    void* dz;                      // row stride lddz (zeros in [M, lddz)), or null
    float* part;                   // [ceil(N / 32)][M], or null
    int64_t ldg, ldz, lddz;
    int dz_dt, strips;             // strips: workgroups side by side along a row
};

// V elements from p
template <int V> __device__ __forceinline__ void load_row(const bf16_t* p, float (&v)[V]) {
    unsigned w[V / 2];
    __builtin_memcpy(w, p, V * 2);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = __uint_as_float(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
}
template <int V> __device__ __forceinline__ void load_row(const float* p, float (&v)[V]) { __builtin_memcpy(v, p, V * 4); }
// `miss` of V values dropped in front, zeros behind (see drop_front)
template <int V> __device__ __forceinline__ void drop_values(float (&v)[V], int miss) {
#pragma unroll
    for (int s = 1; s < V; s *= 2)
        if (miss & s)
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = j + s < V ? v[j + s] : 0.f;
}
// n of V elements of a row shorter than V, zeros behind
template <int V, typename T> __device__ __forceinline__ void load_few(const T* p, int n, float (&v)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = j < n ? Elem<T>::load(p, j) : 0.f;
}

// ZK: SPHIP_F32, SPHIP_BF16, SPHIP_INT8, SPHIP_E4M3, or -1: no activation, z is not read. (The activation as an argument, its
// choice at each of a thread's 32 values, made a kernel four times as long: 256 x 768 9.6 us against 8.4, 4099 x 1500 13.0
// against 11.7.)
template <typename TG, int ZK, int ACT>
__global__ __launch_bounds__(256) void linear_preact_kernel(PreactArgs a, int64_t N, int M) {
    constexpr int V = 16 / sizeof(TG), B = 4;
    constexpr bool CODES = ZK == SPHIP_INT8 || ZK == SPHIP_E4M3;
    __shared__ float red[8][32 * V];
    const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const int64_t grp = blockIdx.x / (unsigned)a.strips, r0 = grp * 32 + rl;
    const int m = ((int)(blockIdx.x % (unsigned)a.strips) * 32 + cl) * V, cols = min(V, M - m);    // <= 0: padding of dz
    const int miss = V - cols;
    float sum[V], v[B][V], z[B][V];
    unsigned q[B][V / 4];
    uint8_t s8[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.f, s8[j] = 0;
    if (CODES && cols > 0) __builtin_memcpy(s8, a.scales + grp * a.ldz + m, V);      // (code rows are padded to 16: whole pieces)
#pragma unroll
    for (int t = 0; t < B; ++t) {
        const int64_t row = r0 + 8 * t;
        const int n = row < N ? cols : 0;
#pragma unroll
        for (int j = 0; j < V; ++j) v[t][j] = z[t][j] = 0.f;
        if (n > 0 && M >= V) {
            load_row<V>((const TG*)a.g + row * a.ldg + m - miss, v[t]);
            if (ZK == SPHIP_F32) load_row<V>((const float*)a.z + row * a.ldz + m - miss, z[t]);
            if (ZK == SPHIP_BF16) load_row<V>((const bf16_t*)a.z + row * a.ldz + m - miss, z[t]);
        } else if (n > 0) {
            load_few<V>((const TG*)a.g + row * a.ldg, n, v[t]);
            if (ZK == SPHIP_F32) load_few<V>((const float*)a.z + row * a.ldz, n, z[t]);
            if (ZK == SPHIP_BF16) load_few<V>((const bf16_t*)a.z + row * a.ldz, n, z[t]);
        }
        if (CODES) {
#pragma unroll
            for (int j = 0; j < V / 4; ++j) q[t][j] = 0;
            if (n > 0) __builtin_memcpy(q[t], (const uint8_t*)a.z + row * a.ldz + m, V);
        }
    }
    if (cols > 0 && miss > 0 && M >= V)
#pragma unroll
        for (int t = 0; t < B; ++t) {
            drop_values<V>(v[t], miss);
            if (ZK == SPHIP_F32 || ZK == SPHIP_BF16) drop_values<V>(z[t], miss);
        }
#pragma unroll
    for (int t = 0; t < B; ++t) {
        const int64_t row = r0 + 8 * t;
        if (CODES) {
#pragma unroll
            for (int j = 0; j < V / 4; ++j) {
                const float s4[4] = {scale_value(s8[4 * j]), scale_value(s8[4 * j + 1]), scale_value(s8[4 * j + 2]), scale_value(s8[4 * j + 3])};
                float o[4];
                code_values<ZK == SPHIP_INT8 ? SPHIP_INT8 : SPHIP_E4M3>(q[t][j], s4, o);
#pragma unroll
                for (int c = 0; c < 4; ++c) z[t][4 * j + c] = o[c];
            }
        }
        if (row >= N) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (ZK >= 0) v[t][j] = j < cols ? v[t][j] * act_slope(z[t][j], ACT) : 0.f;
            sum[j] += v[t][j];
        }
        if (a.dz != nullptr) {
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                const float o[4] = {v[t][j], v[t][j + 1], v[t][j + 2], v[t][j + 3]};
                if (m + j < a.lddz) store4_from_f32(a.dz, a.dz_dt, row * a.lddz + m + j, o);
            }
        }
    }
    if (a.part == nullptr) return;
#pragma unroll
    for (int j = 0; j < V; ++j) red[rl][cl * V + j] = sum[j];
    __syncthreads();
    for (int c = threadIdx.x; c < 32 * V; c += 256) {
        const int col = (int)(blockIdx.x % (unsigned)a.strips) * 32 * V + c;
        if (col >= M) continue;
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) t += red[i][c];
        a.part[grp * M + col] = t;
    }
}

template <typename TG> static int launch_preact(PreactArgs& a, int act, int z_kind, int64_t N, int64_t M, hipStream_t s) {
    constexpr int V = 16 / sizeof(TG);
    const int64_t strips = cdiv(a.dz != nullptr ? a.lddz : M, 32 * V), blocks = cdiv(N, 32) * strips;
    SPHIP_REQUIRE(blocks < MAX_GROUPS, SPHIP_EUNSUPPORTED, "linear_backward: grid too large");
    a.strips = (int)strips;
    const dim3 grid((unsigned)blocks), block(256);
    typedef void (*kern_t)(PreactArgs, int64_t, int);
#define LIN_PREACT(ZK) {linear_preact_kernel<TG, ZK, SPHIP_ACT_RELU>, linear_preact_kernel<TG, ZK, SPHIP_ACT_GELU>, linear_preact_kernel<TG, ZK, SPHIP_ACT_SILU>}
    static const kern_t kerns[4][3] = {LIN_PREACT(SPHIP_F32), LIN_PREACT(SPHIP_BF16), LIN_PREACT(SPHIP_INT8), LIN_PREACT(SPHIP_E4M3)};
#undef LIN_PREACT
    const int zk = z_kind == SPHIP_F32 ? 0 : z_kind == SPHIP_BF16 ? 1 : z_kind == SPHIP_INT8 ? 2 : 3;
    const kern_t fn = act == SPHIP_ACT_NONE ? linear_preact_kernel<TG, -1, SPHIP_ACT_NONE> : kerns[zk][act - SPHIP_ACT_RELU];
    hipLaunchKernelGGL(fn, grid, block, 0, s, a, N, (int)M);
    SPHIP_CHECK_LAUNCH("linear_backward(dz)");
    return SPHIP_OK;
}

// What the products still need after dz, in one launch: the first a.restore workgroups restore x from its codes, the others sum
// 16 columns each of part (P, M), 16 interleaved chains in row order. (Two launches took 3.6 and 3.3 us at 256 x 768 x 768.)
struct FinishArgs {
    RestoreArgs x;
    const float* part;
    void* db;
    int64_t P;
    unsigned restore;
    int M, db_dt;
};
template <typename T, int FMT> __global__ __launch_bounds__(256) void linear_finish_kernel(FinishArgs a) {
    if (blockIdx.x < a.restore) {
        restore_block<T, FMT>(a.x, blockIdx.x);
        return;
    }
    __shared__ float red[16][16];
    const int c = threadIdx.x & 15, w = threadIdx.x >> 4;
    const int m = (int)(blockIdx.x - a.restore) * 16 + c;
    float s = 0.f;
    if (m < a.M)
        for (int64_t p = w; p < a.P; p += 16) s += a.part[p * a.M + m];
    red[w][c] = s;
    __syncthreads();
    if (w == 0 && m < a.M) {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) t += red[j][c];
        store_from_f32(a.db, a.db_dt, m, t);
    }
}
static int launch_finish(FinishArgs& a, int dtype, int fmt, hipStream_t s) {
    const int64_t restore = a.x.codes ? restore_blocks(a.x, dtype) : 0, blocks = restore + (a.db ? cdiv(a.M, 16) : 0);
    SPHIP_REQUIRE(blocks < MAX_GROUPS, SPHIP_EUNSUPPORTED, "linear_backward: grid too large");
    a.restore = (unsigned)restore;
    const dim3 grid((unsigned)blocks), block(256);
    if (dtype == SPHIP_BF16) {
        if (fmt == SPHIP_E4M3) hipLaunchKernelGGL((linear_finish_kernel<bf16_t, SPHIP_E4M3>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((linear_finish_kernel<bf16_t, SPHIP_INT8>), grid, block, 0, s, a);
    } else {
        if (fmt == SPHIP_E4M3) hipLaunchKernelGGL((linear_finish_kernel<float, SPHIP_E4M3>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((linear_finish_kernel<float, SPHIP_INT8>), grid, block, 0, s, a);
    }
    SPHIP_CHECK_LAUNCH("linear_backward(db)");
    return SPHIP_OK;
}

static bool valid_act(int act) { return act >= SPHIP_ACT_NONE && act <= SPHIP_ACT_SILU; }
static bool aligned_elem(const void* p, int dt) { return ((uintptr_t)p & (dtype_size(dt) - 1)) == 0; }

}  // namespace sphip

using namespace sphip;

#define SPHIP_LINEAR_SIZES(what)                                                                                        \
    SPHIP_REQUIRE(N > 0 && D > 0 && M > 0, SPHIP_EINVAL, what ": empty shape N=%lld D=%lld M=%lld", (long long)N,        \
                  (long long)D, (long long)M);                                                                          \
    SPHIP_REQUIRE(N < (1ll << 31) - 256 && D < MAX_LD - 64 && M < MAX_LD - 64, SPHIP_EUNSUPPORTED,                       \
                  what ": N=%lld D=%lld M=%lld: a dimension exceeds int32 (N) or 2^22 features", (long long)N, (long long)D,     \
                  (long long)M)

static bool is_codes(int kind) { return kind == SPHIP_INT8 || kind == SPHIP_E4M3; }
static bool codes_ok(const void* codes, const void* scales, int64_t ld, int64_t cols) {
    return scales && ld >= cols && ld % 16 == 0 && ((uintptr_t)codes & 15) == 0 && ((uintptr_t)scales & 15) == 0;
}
static size_t up256(size_t b) { return (b + 255) / 256 * 256; }

// workspace: partial tiles | z in fp32 on its way into 8 bits | x and W packed (rows that are no whole number of 16 bytes)
struct ForwardSpace {
    size_t part, z, pack, total;
    int copies;
    bool one;
};
// Whether the forward product takes linear_few.hip: one launch, no copies, but its workgroups read all of x each and share K
// among 8 waves only. Its time follows K and the rounds of its workgroups, one per compute unit up to 4096 (or 8192) rows of W;
// the tiles', which also split K, follows W's size. us here / with 64 x 64 tiles, W from HBM (widths around the borders and
// 1700 shapes in all: these rules come within 2 % of the better side on average, 26 % at worst):
//   bf16, up to 8 tokens: 1 x 4096 x 768 6.8 / 7.0, 4096 x 4096 8.6 / 10.8, 8192 x 4096 14.7 / 20.1, 8192 x 768 11.4 / 8.7; 8 x 2048 x
//   8000 9.1 / 11.4, 2048 x 8256 11.7 / 12.6, 4096 x 14336 26.9 / 27.5, but 1024 x 14336 9.5 / 8.6.
//   up to 16: 16 x 3000 x 1000 6.6 / 7.6, 4096 x 4096 10.2 / 11.3, 4096 x 8192 15.5 / 20.6, 4096 x 2048 9.9 / 9.4, 2048 x 8256 13.6 / 12.8.
//   up to 32: 24 x 1536 x 1000 6.1 / 7.5, 2048 x 2048 7.3 / 7.8, 2048 x 6000 9.8 / 12.8, 2048 x 8000 10.1 / 13.0, 2048 x 8192 10.2 / 13.0,
//   4096 x 8000 18.5 / 20.5, but 2048 x 768 7.2 / 7.1, 4096 x 4096 12.6 / 11.5, 2048 x 8256 17.2 / 13.0.
//   fp32, up to 16: 16 x 2048 x 2048 10.2 / 12.0, 4096 x 2048 17.2 / 16.7, 8192 x 4096 36.6 / 46.1, 8192 x 2048 31.6 / 26.5.
//   up to 32: 24 x 1024 x 768 7.4 / 8.6, 2048 x 4096 14.2 / 16.5, 2048 x 2048 13.8 / 12.3; between 4096 and 8192 rows, a round of 32
//   each however few they are: 4096 x 4800 35.8 / 32.7, 4096 x 6000 36.5 / 41.1, 4096 x 8000 40 / 44; 4096 x 9000 68 / 63, 4096 x
//   20000 105 / 135.
//   up to 64: bf16 48 x 512 x 6000 5.5 / 5.8, fp32 48 x 512 x 8000 10.5 / 13.1, but 64 x 1024 x 768 7.1 / 6.8, fp32 11.8 / 8.9.
// Where the tiles would have to copy W or x first (bf16), as long as x is short: 24 x 2049 x 8192 24.9 / 25.8, 40 x 333 x 777
// 7.0 / 8.3, but 48 x 1537 x 3333 22 / 17, 16 x 4097 x 4096 27 / 24.
static bool few(int dtype, int64_t N, int64_t D, int64_t M, int copies) {
    if (N > FEW || (g_forced && g_forced != 'f')) return false;
    if (g_forced) return true;
    const bool bf = dtype == SPHIP_BF16;
    if (copies) return N * D <= 65536;
    if (N > 32) return D <= (bf ? 768 : 512) && M <= 8192;
    if (bf) {
        if (N <= 8) return M > 8192 ? D >= 2048 : D <= 4096 || 2 * M >= D;
        if (M > 8192) return false;
        if (N <= 16) return D <= 3000 || (D <= 4096 && M >= 3000);
        return D <= 1536 || M >= 2 * (D - 1024);
    }
    if (N <= 16) return D <= 2048 || 5 * M >= 2 * D;
    if (D <= 1024) return true;
    return M <= 4096 ? M >= 2 * (D - 1024) : M <= 8192 ? 3 * M >= 2 * 8192 : M > 16384;
}
// Which of the operands have to be copied, for a query and for a launch alike; `odd`: bits of those that are not fetchable().
// Where the rows of x are no whole 16-byte pieces, what follows a row would be multiplied with what follows one of W: both.
enum { COPY_X = 1, COPY_W = 2 };
static int odd_rows(const void* x, int64_t ldx, const void* W, int64_t ldw, int dtype) {
    return (x && !fetchable(x, ldx, (int)dtype_size(dtype)) ? COPY_X : 0) | (W && !fetchable(W, ldw, (int)dtype_size(dtype)) ? COPY_W : 0);
}
static ForwardSpace forward_space(int dtype, int z_kind, int64_t N, int64_t D, int64_t M, int odd) {
    ForwardSpace f;
    f.copies = unaligned(dtype, D) ? COPY_X | COPY_W : odd & (COPY_X | COPY_W);
    f.one = few(dtype, N, D, M, f.copies);
    const bool one = f.one;
    if (one) f.copies = 0;
    f.part = one ? 0 : up256(split_bytes(dtype, N, M, D));
    f.z = is_codes(z_kind) && (f.part || one) ? up256((size_t)N * (cdiv(M, 4) * 4) * 4) : 0;      // (no codes from a split K range or from few rows)
    f.pack = (size_t)((f.copies & COPY_X ? N : 0) + (f.copies & COPY_W ? M : 0)) * packed_ld(D) * dtype_size(dtype);
    f.total = f.part + f.z + f.pack;
    return f;
}
extern "C" size_t sphip_linear_workspace_bytes(int dtype, int z_kind, int64_t N, int64_t D, int64_t M, int odd) {
    if (N <= 0 || D <= 0 || M <= 0 || !valid_dtype(dtype)) return 0;
    read_forced();
    return forward_space(dtype, z_kind, N, D, M, odd).total;
}

extern "C" int sphip_linear(const void* x, int64_t ldx, const void* W, int64_t ldw, int dtype, const void* bias,
                            int bias_dtype, int act, const void* residual, int res_dtype, int64_t ldr, void* out,
                            int out_dtype, int64_t ldo, void* z, int z_kind, uint8_t* z_scales, int64_t ldz, uint8_t* x_codes,
                            uint8_t* x_scales, int x_fmt, int64_t ldq, int64_t N, int64_t D, int64_t M, void* ws,
                            size_t ws_bytes, void* stream) {
    const bool zc = z && is_codes(z_kind);
    SPHIP_REQUIRE(valid_dtype(dtype) && valid_dtype(out_dtype) && (!bias || valid_dtype(bias_dtype)) &&
                      (!residual || valid_dtype(res_dtype)) && (!z || zc || valid_dtype(z_kind)) && (!x_codes || is_codes(x_fmt)),
                  SPHIP_EINVAL, "linear: bad dtype");
    SPHIP_REQUIRE(valid_act(act), SPHIP_EINVAL, "linear: bad activation %d", act);
    SPHIP_REQUIRE(x && W && out, SPHIP_EINVAL, "linear: null pointer");
    SPHIP_LINEAR_SIZES("linear");
    SPHIP_REQUIRE(ldx >= D && ldw >= D && ldo >= M && (!residual || ldr >= M) && (!z || ldz >= M), SPHIP_EINVAL,
                  "linear: a row stride is shorter than its row");
    SPHIP_REQUIRE(aligned_elem(x, dtype) && aligned_elem(W, dtype) && aligned_elem(out, out_dtype) &&
                      (!bias || aligned_elem(bias, bias_dtype)) && (!residual || aligned_elem(residual, res_dtype)) &&
                      (!z || zc || aligned_elem(z, z_kind)),
                  SPHIP_EINVAL, "linear: a pointer is not aligned to its element");
    SPHIP_REQUIRE((!zc || codes_ok(z, z_scales, ldz, M)) && (!x_codes || codes_ok(x_codes, x_scales, ldq, D)), SPHIP_EINVAL,
                  "linear: codes and scales need 16-byte aligned rows of at least their columns");
    read_forced();
    const ForwardSpace f = forward_space(dtype, zc ? z_kind : SPHIP_F32, N, D, M, odd_rows(x, ldx, W, ldw, dtype));
    SPHIP_REQUIRE(f.total == 0 || (ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= f.total), SPHIP_EWORKSPACE,
                  "linear: workspace of %zu bytes, needs %zu, 16-byte aligned", ws_bytes, f.total);
    hipStream_t s = (hipStream_t)stream;
    Epilogue e;
    e.bias = bias, e.bias_dt = bias_dtype, e.res = residual, e.res_dt = res_dtype, e.ldr = ldr;
    e.out = out, e.out_dt = out_dtype, e.ldo = ldo, e.act = act;
    // z becomes codes in the epilogue itself, unless the K range is split: its partial sums then meet in the joining kernel,
    // which has no groups of rows (nor has the kernel for few rows), and z takes the way over fp32
    if (zc && f.z) e.z = (char*)ws + f.part, e.z_dt = SPHIP_F32, e.ldz = cdiv(M, 4) * 4;
    else e.z = z, e.z_dt = z_kind, e.ldz = ldz, e.z_scales = zc ? z_scales : nullptr;
    Operand A = {x, ldx, (int)N}, B = {W, ldw, (int)M};
    // K up to whole pieces only where zeros follow the rows of both operands: behind the rows of one that is not copied lies
    // the next row, or the end of its memory (fp32 copies one alone, whatever D is; bf16 with such a D copies both)
    const int64_t K = f.copies == (COPY_X | COPY_W) ? whole_pieces(D) : D, ld = packed_ld(D);
    char* to = (char*)ws + f.part + f.z;
    int st = SPHIP_OK;
    Packing p(dtype);
    if (x_codes) {                                              // x is read once for its codes and its copy
        const bool copy = f.copies & COPY_X;
        st = save_codes("linear", x, dtype, ldx, x_fmt, 0, x_codes, x_scales, ldq, copy ? to : nullptr, copy ? ld : 0, N, D, s);
        if (copy) A.p = to, A.ld = ld;
    } else if (f.copies & COPY_X) {
        p.add(A, N, D, to);
    }
    if (f.copies & COPY_W) p.add(B, M, D, to + (f.copies & COPY_X ? (size_t)N * ld * dtype_size(dtype) : 0));
    if (st == SPHIP_OK) st = p.launch("linear", s);
    if (st != SPHIP_OK) return st;
    st = f.one ? launch_linear_few("linear", dtype, A, B, e, K, s)
         : dtype == SPHIP_BF16 ? launch_product<bf16_t, OP_ROWS, OP_ROWS>("linear", A, B, e, K, K, ws, f.part, s)
                               : launch_product<float, OP_ROWS, OP_ROWS>("linear", A, B, e, K, K, ws, f.part, s);
    if (st == SPHIP_OK && zc && f.z)
        st = save_codes("linear", e.z, SPHIP_F32, e.ldz, z_kind, act == SPHIP_ACT_RELU, (uint8_t*)z, z_scales, ldz, nullptr, 0, N, M, s);
    return st;
}

// workspace: dz | column sums of 32-row groups | x as aligned rows (restored from codes, or packed) | W packed | partial tiles
// of a product
struct BackwardSpace {
    size_t dz, sums, x, w, part, total;
};
static BackwardSpace backward_space(int dtype, int x_kind, int want_dx, int want_dw, int want_db, int64_t N, int64_t D, int64_t M,
                                    int odd) {
    BackwardSpace b;
    const size_t es = dtype_size(dtype);
    b.dz = want_dx || want_dw ? up256((size_t)N * packed_ld(M) * es) : 0;
    b.sums = want_db ? up256((size_t)cdiv(N, 32) * M * 4) : 0;
    b.x = want_dw && (is_codes(x_kind) || (odd & COPY_X)) ? up256((size_t)N * packed_ld(D) * es) : 0;
    b.w = want_dx && (odd & COPY_W) ? up256((size_t)M * packed_ld(D) * es) : 0;
    const size_t p1 = want_dx ? split_bytes(dtype, N, D, M) : 0, p2 = want_dw ? split_bytes(dtype, M, D, N) : 0;
    b.part = p1 > p2 ? p1 : p2;
    b.total = b.dz + b.sums + b.x + b.w + b.part;
    return b;
}

extern "C" size_t sphip_linear_backward_workspace_bytes(int dtype, int x_kind, int want_dx, int want_dw, int want_db, int64_t N,
                                                        int64_t D, int64_t M, int odd) {
    if (N <= 0 || D <= 0 || M <= 0 || !valid_dtype(dtype)) return 0;
    read_forced();
    return backward_space(dtype, x_kind, want_dx, want_dw, want_db, N, D, M, odd).total;
}

extern "C" int sphip_linear_backward(const void* g, int g_dtype, int64_t ldg, const void* W, int64_t ldw, int dtype, int act,
                                     const void* z, int z_kind, const uint8_t* z_scales, int64_t ldz, const void* x, int x_kind,
                                     const uint8_t* x_scales, int64_t ldx, void* dx, int dx_dtype, int64_t lddx, void* dW,
                                     int dw_dtype, int64_t lddw, void* db, int db_dtype, int64_t N, int64_t D, int64_t M,
                                     void* ws, size_t ws_bytes, void* stream) {
    SPHIP_REQUIRE(valid_dtype(dtype) && valid_dtype(g_dtype) && (!dx || valid_dtype(dx_dtype)) && (!dW || valid_dtype(dw_dtype)) &&
                      (!db || valid_dtype(db_dtype)),
                  SPHIP_EINVAL, "linear_backward: bad dtype");
    SPHIP_REQUIRE(valid_act(act), SPHIP_EINVAL, "linear_backward: bad activation %d", act);
    SPHIP_LINEAR_SIZES("linear_backward");
    SPHIP_REQUIRE(g && (dx || dW || db) && (!dx || W) && (!dW || x), SPHIP_EINVAL, "linear_backward: null pointer");
    const bool zc = is_codes(z_kind), xc = is_codes(x_kind);
    SPHIP_REQUIRE(act == SPHIP_ACT_NONE || (z && (zc || valid_dtype(z_kind))), SPHIP_EINVAL,
                  "linear_backward: an activation needs z (values, or codes with scales)");
    SPHIP_REQUIRE(!dW || xc || x_kind == dtype, SPHIP_EINVAL, "linear_backward: x must be of the product's type or 8-bit codes");
    SPHIP_REQUIRE(ldg >= M && (!dx || (ldw >= D && lddx >= D)) && (!dW || (ldx >= D && lddw >= D)) &&
                      (act == SPHIP_ACT_NONE || ldz >= M),
                  SPHIP_EINVAL, "linear_backward: a row stride is shorter than its row");
    SPHIP_REQUIRE((act == SPHIP_ACT_NONE || !zc || codes_ok(z, z_scales, ldz, M)) && (!dW || !xc || codes_ok(x, x_scales, ldx, D)),
                  SPHIP_EINVAL, "linear_backward: codes and scales need 16-byte aligned rows of at least their columns");
    SPHIP_REQUIRE(aligned_elem(g, g_dtype) && (!dx || (aligned_elem(W, dtype) && aligned_elem(dx, dx_dtype))) &&
                      (!dW || ((xc || aligned_elem(x, dtype)) && aligned_elem(dW, dw_dtype))) && (!db || aligned_elem(db, db_dtype)) &&
                      (act == SPHIP_ACT_NONE || zc || aligned_elem(z, z_kind)),
                  SPHIP_EINVAL, "linear_backward: a pointer is not aligned to its element");
    read_forced();
    const BackwardSpace sp = backward_space(dtype, x_kind, dx != nullptr, dW != nullptr, db != nullptr, N, D, M,
                                            odd_rows(xc || !dW ? nullptr : x, ldx, dx ? W : nullptr, ldw, dtype));
    SPHIP_REQUIRE(sp.total == 0 || (ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= sp.total), SPHIP_EWORKSPACE,
                  "linear_backward: workspace of %zu bytes, needs %zu, 16-byte aligned", ws_bytes, sp.total);
    hipStream_t s = (hipStream_t)stream;
    char* w = (char*)ws;
    float* sums = (float*)(w + sp.dz);
    // Without an activation the incoming gradient is dz. It is copied (into the product's dtype, rows padded to 64) only
    // where it does not have that dtype, or where LDS-DMA could not fetch it as it is.
    const bool products = dx || dW;
    const bool direct = act == SPHIP_ACT_NONE && g_dtype == dtype && fetchable(g, ldg, (int)dtype_size(dtype)) && !(dx && unaligned(dtype, M));
    Operand dz = {g, ldg, (int)N}, ow = {W, ldw, (int)D}, ox = {x, ldx, (int)D};
    Packing pack(dtype);
    const bool copied = products && !direct && !db && act == SPHIP_ACT_NONE && g_dtype == dtype;
    if (copied) pack.add(dz, N, M, w);                          // g with padded rows is all there is to do
    else if (products && !direct) dz.p = w, dz.ld = packed_ld(M);
    char *const xs = w + sp.dz + sp.sums, *const part = xs + sp.x + sp.w;
    if (sp.w) pack.add(ow, M, D, xs + sp.x);
    if (sp.x && !xc) pack.add(ox, N, D, xs);
    int st = pack.launch("linear_backward", s);
    if (st != SPHIP_OK) return st;
    if (!copied && (db || (products && !direct))) {
        PreactArgs a;
        a.g = g, a.z = z, a.scales = z_scales, a.dz = products && !direct ? w : nullptr, a.part = db ? sums : nullptr;
        a.ldg = ldg, a.ldz = ldz, a.lddz = dz.ld, a.dz_dt = dtype;
        st = g_dtype == SPHIP_BF16 ? launch_preact<bf16_t>(a, act, z_kind, N, M, s) : launch_preact<float>(a, act, z_kind, N, M, s);
        if (st != SPHIP_OK) return st;
    }
    if (db || (dW && xc)) {
        FinishArgs a = {};
        if (dW && xc) {
            a.x = {(const uint8_t*)x, x_scales, xs, ldx, packed_ld(D), N, (int)D};
            ox.p = xs, ox.ld = a.x.ldo;
        }
        a.part = sums, a.db = db, a.P = cdiv(N, 32), a.M = (int)M, a.db_dt = db_dtype;
        st = launch_finish(a, dtype, x_kind, s);
        if (st != SPHIP_OK) return st;
    }
    Epilogue e;
    if (dx) {
        e.out = dx, e.out_dt = dx_dtype, e.ldo = lddx;
        const int64_t K = direct ? M : whole_pieces(M);         // (dz is padded with zeros)
        st = dtype == SPHIP_BF16 ? launch_product<bf16_t, OP_ROWS, OP_COLS>("linear_backward(dx)", dz, ow, e, K, M, part, sp.part, s)
                                 : launch_product<float, OP_ROWS, OP_COLS>("linear_backward(dx)", dz, ow, e, K, M, part, sp.part, s);
        if (st != SPHIP_OK) return st;
    }
    if (dW) {
        e.out = dW, e.out_dt = dw_dtype, e.ldo = lddw;
        dz.rows = (int)M;
        st = dtype == SPHIP_BF16 ? launch_product<bf16_t, OP_COLS, OP_COLS>("linear_backward(dW)", dz, ox, e, N, N, part, sp.part, s)
                                 : launch_product<float, OP_COLS, OP_COLS>("linear_backward(dW)", dz, ox, e, N, N, part, sp.part, s);
    }
    return st;
}
