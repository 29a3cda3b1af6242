// gemm_f8.hip -- products of 8-bit floating point with a scale for each block of 128:
//   y[r, c] = sum_b sx[r, b] sw[c / 128, b] sum_{k in block b} x[r, k] w[c, k].
//
// A block's sum is formed by the matrix cores and added to y in f32 with both scales: weights are the first operand, so a lane holds four neighbouring columns of
// one row, whose scale is the lane's own; the columns' scale is the same for a whole tile.
//
// Which matrix instruction.  v_mfma_f32_16x16x128_f8f6f4 takes 128 products at once, but adds them up eight at a time with the products aligned to the largest one's power
// of two and cut off 2^-13 below it (measured: 1.4e-5 of the results' size for operands of one size, whatever the number of blocks, up to 6e-5 where columns are powers of ten apart),
// where f32 sums keep 1e-7.  f16 results are rounded by 2.1e-4 of their size anyway.  So it is taken for f16 results of more than 16 rows (GEMM_F8_EXACT: not there either).  Fewer
// are bound by memory, and f32 results are to be as exact as f32 is: there the codes become f16 numbers (exactly: one conversion per pair) for v_mfma_f32_16x16x32_f16.
//
// Measured, with the conversion of f16 or f32 rows: 1 row of 4096 x 4096 5.4 us; 16 rows of 32000 x 4096, f32 results, 29.8 us, the weights at 5.5 TB/s in 24 of it; 64 rows of 11008 x 4096
// 16.3 us; 131 rows of 4096 x 11008, f32 results, 30 us; 2048 rows of 13824 x 5120 from 8 bits 152 us, 1.9 PFLOP/s (a library product with one scale for all: 116 us).
#include "kernels.h"
#include "answers.h"
#include "q4.h"

#include <algorithm>

namespace rlh {

typedef __attribute__((ext_vector_type(8))) int int8_t_;
typedef __amdgpu_buffer_rsrc_t buffer_t;

__device__ __forceinline__ buffer_t f8_buffer(const void *data, size_t offset, size_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(reinterpret_cast<const char *>(data)) + offset, 0, (int)bytes, 0x00027000);
}
constexpr int kF8Outside = 0x7ffffff0; // an offset past every buffer: reads as zeros

// sixteen codes as two operands of the f16 instruction
__device__ __forceinline__ half8_t f8_half8(uint32_t a, uint32_t b) {
    const half2_t x0 = f8_pair_f16<false>(a), x1 = f8_pair_f16<true>(a), x2 = f8_pair_f16<false>(b), x3 = f8_pair_f16<true>(b);
    return half8_t{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
}

// Columns n .. n + 3 of a row, of which `left` are inside.  (Rows of any length: the element's alignment is enough for one store.  One by one where rows are no multiple of four
// columns: 1064 x 4959 x 496 23.1 us, 18.7 so; 865 x 333 x 10304 in f32 39 and 32.)
template <typename Y>
__device__ __forceinline__ void store_row4(Y *y, int n, int left, const float4_t &v) {
    typedef Y any __attribute__((ext_vector_type(4), aligned(sizeof(Y))));
    if (left >= 4) {
        *reinterpret_cast<any *>(y + n) = any{(Y)v[0], (Y)v[1], (Y)v[2], (Y)v[3]};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < left) y[n + i] = (Y)v[i];
}

// ---- few rows --------------------------------------------------------------------------------------------------------------------------
// Up to 16 rows.  A workgroup owns all of them and 16 kNF columns; its wavefronts share the blocks of K, each reading its operands from memory into registers and
// nowhere else, and add their sums up through LDS in their own order.
//
// A few rows of f16 or f32 are converted by the workgroup itself: a wavefront converts the blocks that it needs, sixteen lanes a row's block, while its first
// weights are on their way, and keeps the codes in LDS.  (A launch of its own took 5 us; converted by the lanes that use them, sixteen times over for one row, 3 us.)
enum F8Source { kF8Codes = 0, kF8FromF16 = 1, kF8FromF32 = 2 };
struct RowsF8Params {
    MatmulF8Params p;
    const void *src; // f16 or f32 rows, converted on the way
};
constexpr int kRfLds = 96 * 1024; // for converted rows

template <int kNF, int kSource, typename Y>
__global__ __launch_bounds__(kRfWaves *kWave) void matmul_f8_rows_kernel(RowsF8Params pp) {
    const MatmulF8Params &p = pp.p;
    constexpr int kScales = kF8Block % (16 * kNF) == 0 ? 1 : kNF; // of the workgroup's columns
    __shared__ __attribute__((aligned(16))) float4_t red[kRfWaves][kNF][kWave];
    extern __shared__ __attribute__((aligned(16))) unsigned char converted[]; // of each wavefront the codes [block][row][128], then the scales
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int c = lane & 15, h = lane >> 4;
    const int n0 = blockIdx.x * 16 * kNF, across = f8_blocks(p.k);
    const int rows_w = min(p.n - n0, 16 * kNF);
    const buffer_t wb = f8_buffer(p.w.codes, (size_t)n0 * p.k, (size_t)rows_w * p.k);
    const buffer_t xb = f8_buffer(p.x.codes, 0, (size_t)p.m * p.k);
    const buffer_t sb = f8_buffer(p.x.scales, 0, (size_t)p.m * across * 4);
    int w_at[kNF];
#pragma unroll
    for (int j = 0; j < kNF; j++) w_at[j] = min(j * 16 + c, rows_w - 1) * p.k + h * 16;
    const int my_row = min(c, p.m - 1), x_at = my_row * p.k + h * 16, s_at = my_row * across * 4;
    struct Block {
        uint32_t w[kNF][8], x[8];
        float sx, sw[kScales];
    };
    auto take = [](uint32_t *to, buffer_t from, int at) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b128(from, at, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; i++) to[i] = v[i];
    };
    auto load = [&](Block &k, int b) __attribute__((always_inline)) {
        const int k0 = b * kF8Block;
        // a lane's 32 bytes of a block are pieces h and h + 4: each load takes whole halves of lines
        const bool in0 = k0 + h * 16 < p.k, in1 = k0 + h * 16 + 64 < p.k;
#pragma unroll
        for (int j = 0; j < kNF; j++) {
            take(k.w[j], wb, in0 ? w_at[j] + k0 : kF8Outside);
            take(k.w[j] + 4, wb, in1 ? w_at[j] + k0 + 64 : kF8Outside);
        }
        if constexpr (kSource == kF8Codes) {
            take(k.x, xb, in0 ? x_at + k0 : kF8Outside);
            take(k.x + 4, xb, in1 ? x_at + k0 + 64 : kF8Outside);
            k.sx = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(sb, s_at + b * 4, 0, 0));
        }
#pragma unroll
        for (int t = 0; t < kScales; t++) k.sw[t] = p.w.scales[(size_t)(min(n0 + t * 16, p.n - 1) / kF8Block) * across + b];
    };
    // Workgroups in step would ask for the same columns of all rows, which meet in few memory channels: each starts at another block.
    const int rot = (int)(blockIdx.x * 5u % (unsigned)across);
    auto block_of = [&](int t) {
        const int b = t + rot;
        return b < across ? b : b - across;
    };
    // converted rows: the wavefront's block t is its t / 8-th
    const int share = rows_f8_share(p.k);
    unsigned char *const codes = converted + wave * rows_f8_region(p.m, p.k);
    float *const scales = reinterpret_cast<float *>(codes + (size_t)share * p.m * kRfRow);
    Block now, next;
    if constexpr (kSource == kF8Codes) {
        if (wave < across) load(now, block_of(wave));
    } else {
        constexpr int kBytes = kSource == kF8FromF16 ? 2 : 4, kLoads = kBytes / 2, kBatch = 4;
        const buffer_t src = f8_buffer(pp.src, 0, (size_t)p.m * p.k * kBytes);
        const int mine = across > wave ? (across - wave + kRfWaves - 1) / kRfWaves : 0, items = mine * p.m; // (block, row), four at a time
        for (int first = 0; first < items; first += 4 * kBatch) {
            uint32_t raw[kBatch][4 * kLoads];
#pragma unroll
            for (int u = 0; u < kBatch; u++) {
                const int item = first + u * 4 + h, t = item / p.m, r = item - t * p.m, k0 = block_of(min(wave + t * kRfWaves, across - 1)) * kF8Block + c * 8;
                const int at = item < items && k0 < p.k ? (r * p.k + k0) * kBytes : kF8Outside;
#pragma unroll
                for (int l = 0; l < kLoads; l++) take(raw[u] + 4 * l, src, at == kF8Outside ? at : at + 16 * l);
            }
            if (first == 0) load(now, block_of(wave));
#pragma unroll
            for (int u = 0; u < kBatch; u++) {
                const int item = first + u * 4 + h;
                float v[8], top = 0.0f, odd = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    v[e] = kSource == kF8FromF16 ? (float)__builtin_bit_cast(half2_t, raw[u][e / 2])[e % 2] : __builtin_bit_cast(float, raw[u][e % (4 * kLoads)]);
                    top = fmaxf(top, fabsf(v[e]));
                    odd = fmaf(v[e], 0.0f, odd);
                }
                top = fmaxf(top, quad_perm<kDppQuadPerm1032>(top)); // over the sixteen lanes of the block
                top = fmaxf(top, quad_perm<kDppQuadPerm2301>(top));
                top = fmaxf(top, quad_perm<kDppRowHalfMirror>(top));
                top = fmaxf(top, quad_perm<kDppRowMirror>(top));
                odd = group_sum<16>(odd);
                const F8Scale by(top);
                typedef __attribute__((ext_vector_type(2))) uint32_t uint2_t;
                uint2_t w;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int lo = f8_codes<false>(v[4 * e] * by.factor, v[4 * e + 1] * by.factor, 0);
                    w[e] = (uint32_t)f8_codes<true>(v[4 * e + 2] * by.factor, v[4 * e + 3] * by.factor, lo);
                }
                if (item < items) {
                    *reinterpret_cast<uint2_t *>(codes + (size_t)item * kRfRow + c * 8) = w;
                    if (c == 0) scales[item] = odd == 0.0f ? by.scale : NAN;
                }
            }
        }
        // (a wavefront reads back only what it wrote)
    }
    float4_t acc[kNF];
#pragma unroll
    for (int j = 0; j < kNF; j++) acc[j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    auto use = [&](Block &k, int t) __attribute__((always_inline)) {
        if constexpr (kSource != kF8Codes) {
            const int item = t / kRfWaves * p.m + my_row;
            const uint4_t lo = *reinterpret_cast<const uint4_t *>(codes + (size_t)item * kRfRow + h * 16), hi = *reinterpret_cast<const uint4_t *>(codes + (size_t)item * kRfRow + h * 16 + 64);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                k.x[i] = lo[i];
                k.x[4 + i] = hi[i];
            }
            k.sx = scales[item];
        }
        half8_t xs[4];
#pragma unroll
        for (int q = 0; q < 4; q++) xs[q] = f8_half8(k.x[2 * q], k.x[2 * q + 1]);
#pragma unroll
        for (int j = 0; j < kNF; j++) {
            float4_t part = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int q = 0; q < 4; q++) part = __builtin_amdgcn_mfma_f32_16x16x32_f16(f8_half8(k.w[j][2 * q], k.w[j][2 * q + 1]), xs[q], part, 0, 0, 0);
            const float by = k.sx * k.sw[kScales > 1 ? j : 0];
#pragma unroll
            for (int e = 0; e < 4; e++) acc[j][e] = fmaf(part[e], by, acc[j][e]);
        }
    };
    for (int t = wave; t < across; t += kRfWaves) {
        if (t + kRfWaves < across) load(next, block_of(t + kRfWaves));
        use(now, t);
        now = next;
    }
#pragma unroll
    for (int j = 0; j < kNF; j++) red[wave][j][lane] = acc[j];
    __syncthreads();
    Y *y = reinterpret_cast<Y *>(p.y);
    for (int s = tid; s < kNF * kWave; s += kRfWaves * kWave) {
        const int f = s / kWave, l = s % kWave, r = l & 15, n = n0 + f * 16 + (l >> 4) * 4;
        float4_t v = red[0][f][l];
#pragma unroll
        for (int w = 1; w < kRfWaves; w++) v += red[w][f][l];
        if (r < p.m && n < p.n) store_row4(y + (size_t)r * p.n, n, p.n - n, v);
    }
}

// ---- many rows -------------------------------------------------------------------------------------------------------------------------
// A workgroup owns 16 kMT kWM rows and 16 kNT kWN columns; blocks of K pass by in kStages LDS stages of 128 bytes of every row.  A wavefront keeps its rows' operands of a
// block and reads those of its columns two tiles ahead.  The one barrier of a block comes before its last two column tiles: by then everybody has read the whole stage, so
// the loads of the block kStages further on go there, and the next block, on its way for kStages - 1 blocks, has landed; its first operands are read
// beside the last products, and the matrix cores do not wait between blocks.  (A barrier between blocks left them idle for 700 of 3300 cycles.)  Behind the last block
// the last one is loaded again, so that every block waits for the same number of loads and has no branches, which would pull the products apart.
//
// LDS places.  Sixteen-byte pieces of a row are permuted by (row / 2) % 8, and a lane's 32 bytes of K are pieces h and h + 4: the lanes that an LDS read serves at once (0 .. 3, 12 .. 15
// and 20 .. 27, for instance) are then in 16 different places.  With pieces 2 h and 2 h + 1 they met two by two.
// The rows' scales come through LDS as well: a lane that reads its own from memory touches a line of its own.  With many stages by a load of four bytes per row beside each
// block's; with two, in large tiles, eight blocks at a time through registers (2048 x 13824 x 5120: 169 us with a load per block, 151 so).
__device__ const uint4_t f8_zeros = {0u, 0u, 0u, 0u};

struct TilesF8Params {
    MatmulF8Params p;
    float *parts;  // [pieces x m x n] sums of ranges of blocks, or null: y itself
    int pieces;
    int tiles_m, tiles_n;
};

// (Two wavefronts to a SIMD where LDS, 80 KB of it, leaves room for two workgroups: 256 registers, and the products' results are where the vector ALU reads them.  With more the
// compiler moves each through another register: 64 x 11008 x 4096 19.3 us, 18.4 so.)
template <int kWM, int kWN, int kMT, int kNT, int kStages, bool kExact, typename Y>
__global__ __launch_bounds__(kWM *kWN *kWave, kWM * kWN == 8 || kStages * (kMT * kWM + kNT * kWN) * 16 <= 640 ? 2 : 1) void matmul_f8_tiles_kernel(TilesF8Params pp) {
    const MatmulF8Params &p = pp.p;
    constexpr int kWaves = kWM * kWN, kBM = 16 * kMT * kWM, kBN = 16 * kNT * kWN, kTiles = kMT * kNT;
    constexpr int kStageBytes = (kBM + kBN) * kF8Block;
    constexpr int kLoads = kStageBytes / 1024 / kWaves;         // of a wavefront, eight rows each
    constexpr int kRing = 4, kAhead = 2;                        // operands of columns: places, and how far ahead they are read
    constexpr int kMeet = (kNT - kAhead) * kMT;                 // the tile before which the barrier is
    constexpr int kChunks = (kBM + 63) / 64;                    // of rows whose scales a wavefront-wide load takes; one more is the columns'
    constexpr int kWT = (kBN + kF8Block - 1) / kF8Block;        // tiles of weights' scales side by side
    static_assert(128 % (16 * kNT) == 0, "a wavefront's columns share their scale");
    constexpr int kLoadsX = kBM / 8 / kWaves;
    static_assert(kBM % (8 * kWaves) == 0 && kBN % (8 * kWaves) == 0, "whole loads of every wavefront, of x and then of w");
    static_assert(kNT % kRing == 0 && kNT >= kRing && kRing % 2 == 0, "a block's first column has the same place as the one before it");
    static_assert(kChunks + 1 <= kWaves, "a wavefront for each chunk of scales");
    constexpr bool kSpans = kStages == 2;                       // scales of kSpan blocks at a time
    constexpr int kSpan = 8, kScales = kBM * kSpan / (kWaves * kWave), kExtra = kSpans ? 0 : 1; // a thread's share of them; loads of scales beside a block's
    static_assert(!kSpans || (kBM * kSpan % (kWaves * kWave) == 0 && kSpan % kScales == 0), "a thread's scales are of one row");
    static_assert((kStages - 1) * (kLoads + kExtra) < 64, "loads that are counted");
    __shared__ __attribute__((aligned(1024))) unsigned char lds[kStages * kStageBytes];
    __shared__ __attribute__((aligned(256))) float scales_lds[kSpans ? 2 * kSpan : kStages][kChunks + 1][64];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int c = lane & 15, h = lane >> 4, wm = wave / kWN, wn = wave % kWN;
    const int across = f8_blocks(p.k);
    const int piece = blockIdx.y, b0 = (int)((int64_t)across * piece / pp.pieces), b1 = (int)((int64_t)across * (piece + 1) / pp.pieces);
    // Workgroups of one XCD, eight apart, take tiles that lie together: all rows of a stretch of columns, row tiles first.
    const int tiles = pp.tiles_m * pp.tiles_n, xcd = blockIdx.x % 8;
    const int tile = (int)((int64_t)tiles * xcd / 8) + (int)(blockIdx.x / 8);
    if (tile >= (int)((int64_t)tiles * (xcd + 1) / 8)) return;
    const int tm = tile % pp.tiles_m, tn = tile / pp.tiles_m;
    const int m0 = tm * kBM, n0 = tn * kBN;
    const unsigned lds_base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) void *)lds;

    // staging: rows of x, then of w; a wavefront-wide load covers eight rows, and the sixteen bytes of a lane are those that belong in its place
    const uint8_t *x0 = p.x.codes + (size_t)m0 * p.k, *w0 = p.w.codes + (size_t)n0 * p.k;
    asm volatile("" : "+s"(x0), "+s"(w0)); // (kept in scalar registers, which the loads take them from)
    uint32_t from[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
        const int r = (i * kWaves + wave) * 8 + lane / 8; // row of the stage
        const int row = i < kLoadsX ? min(r, p.m - 1 - m0) : min(r - kBM, p.n - 1 - n0);
        from[i] = (uint32_t)row * (uint32_t)p.k + (uint32_t)((lane % 8) ^ ((r >> 1) & 7)) * 16u; // (below 2^32: 256 rows of 2^24)
    }
    // a wavefront's load of scales: rows 64 chunk + lane, or the columns' tiles
    const int chunk = wave < kChunks ? wave : wave % (kChunks + 1);
    const float *s0 = chunk < kChunks ? p.x.scales + (size_t)m0 * across : p.w.scales + (size_t)(n0 / kF8Block) * across;
    asm volatile("" : "+s"(s0));
    const uint32_t s_from = (uint32_t)(chunk < kChunks ? min(chunk * 64 + lane, p.m - 1 - m0) : min(min(lane, kWT - 1), (p.n - 1) / kF8Block - n0 / kF8Block)) * (uint32_t)across * 4u;
    const unsigned s_base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) void *)scales_lds + (unsigned)chunk * 256u;
    // spans: a thread has kScales neighbouring blocks of one row, the first ones one of a column tile
    const int sp_row = kSpans ? tid / (kSpan / kScales) : 0, sp_block = kSpans ? tid % (kSpan / kScales) * kScales : 0;
    const float *const sp_from = p.x.scales + (size_t)min(m0 + sp_row, p.m - 1) * across, *const sp_from_w = p.w.scales + (size_t)min(n0 / kF8Block + tid / kSpan % kWT, (p.n - 1) / kF8Block) * across;
    float sp_held[kSpans ? kScales : 1], sp_held_w = 0.0f;
    // The blocks in their order: one behind the last whole block of a row goes first.  Load i of the t-th block; kLoads is that of the scales.
    const int whole = p.k / kF8Block, count = b1 - b0, short_first = b1 > whole ? 1 : 0;
    auto block_at = [&](int t) { return t < short_first ? whole : b0 + t - short_first; };
    auto fetch1 = [&](int b, int t, int i) __attribute__((always_inline)) {
        const unsigned stage = (unsigned)t % kStages;
        if (i < kLoads) dma16_base(reinterpret_cast<const half_t *>((i < kLoadsX ? x0 : w0) + (size_t)b * kF8Block), from[i < kLoads ? i : 0], lds_base + stage * kStageBytes + (unsigned)(i * kWaves + wave) * 1024u);
        else dma4_base(s0 + b, s_from, s_base + stage * (unsigned)((kChunks + 1) * 256));
    };
    auto take_span = [&](int span) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kScales; i++) sp_held[i] = sp_from[block_at(min(span * kSpan + sp_block + i, count - 1))];
        sp_held_w = sp_from_w[block_at(min(span * kSpan + tid % kSpan, count - 1))];
    };
    auto put_span = [&](int span) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kScales; i++) scales_lds[(span & 1) * kSpan + sp_block + i][0][sp_row] = sp_held[i];
        if (tid < kSpan * kWT) scales_lds[(span & 1) * kSpan + tid % kSpan][kChunks][tid / kSpan] = sp_held_w;
    };
    auto fetch = [&](int t) __attribute__((always_inline)) { // the t-th block, or the last one again
        const int b = block_at(min(t, count - 1));
        if (b < whole) {
#pragma unroll
            for (int i = 0; i < kLoads + kExtra; i++) fetch1(b, t, i);
            return;
        }
        int l = lane; // columns b * 128 .. of rows whose length is no multiple of 128: zeros behind them
        asm volatile("" : "+v"(l)); // (worked out here: kept in registers through the loop it cost more than 16 of them)
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const int r = (i * kWaves + wave) * 8 + l / 8, at = ((l % 8) ^ ((r >> 1) & 7)) * 16;
            const uint8_t *row = i < kLoadsX ? x0 + (size_t)min(r, p.m - 1 - m0) * p.k : w0 + (size_t)min(r - kBM, p.n - 1 - n0) * p.k;
            const uint8_t *from16 = b * kF8Block + at < p.k ? row + (size_t)b * kF8Block + at : reinterpret_cast<const uint8_t *>(&f8_zeros);
            dma16(reinterpret_cast<const half_t *>(from16), lds_base + ((unsigned)t % kStages) * kStageBytes + (unsigned)(i * kWaves + wave) * 1024u);
        }
        if (!kSpans) fetch1(b, t, kLoads);
    };
    const int nw = n0 + wn * kNT * 16; // the wavefront's first column
    float4_t acc[kMT][kNT];
#pragma unroll
    for (int i = 0; i < kMT; i++)
#pragma unroll
        for (int j = 0; j < kNT; j++) acc[i][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    const unsigned char *const frag_x = lds + (wm * kMT * 16 + c) * kF8Block, *const frag_w = lds + (kBM + wn * kNT * 16 + c) * kF8Block;
    const int p0 = (h ^ (c >> 1)) << 4, p1 = ((h + 4) ^ (c >> 1)) << 4;
    auto frag = [&](const unsigned char *at, int f, int t, uint32_t (&to)[8]) __attribute__((always_inline)) {
        at += ((unsigned)t % kStages) * kStageBytes + f * (16 * kF8Block);
        const uint4_t lo = *reinterpret_cast<const uint4_t *>(at + p0), hi = *reinterpret_cast<const uint4_t *>(at + p1);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            to[i] = lo[i];
            to[4 + i] = hi[i];
        }
    };
    uint32_t x[kMT][8], w[kRing][8];
    float scale[kMT], sx_next[kMT], sw_next;
    auto read_scales = [&](int t) __attribute__((always_inline)) {
        const float *at = scales_lds[(unsigned)t % (kSpans ? 2 * kSpan : kStages)][0];
        sw_next = at[kChunks * 64 + wn * kNT * 16 / kF8Block];
#pragma unroll
        for (int i = 0; i < kMT; i++) sx_next[i] = at[(wm * kMT + i) * 16 + c];
    };
    auto meet = [&](auto left) __attribute__((always_inline)) { // all but `left` loads, and the reads, of this wavefront are done, and behind the barrier everybody's
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt<decltype(left)::value>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    constexpr std::integral_constant<int, (kStages - 2) * (kLoads + kExtra)> kOnTheWay{};
    // kExact: operands as f16 numbers, converted between the products that come before the ones that take them first: a row's beside the first column, a column's a part
    // beside each tile of the column before it.  The four products of a tile wait for each other, and a wavefront issues in order: so everything else stands between them.
    // (All rows' conversions in front of a block's first product, a column's in front of its own, sums behind a tile's four products: 131 x 4096 x 11008 33 us, 31 so; 64 x 11008 x 4096 19.8, 18.4.)
    half8_t xs[kExact ? kMT : 1][4], ws[kExact ? 2 : 1][4];
    auto row_f16 = [&](int i, int q) __attribute__((always_inline)) { xs[i][q] = f8_half8(x[i][2 * q], x[i][2 * q + 1]); };
    auto column_f16 = [&](int j, int q) __attribute__((always_inline)) { ws[j % 2][q] = f8_half8(w[j % kRing][2 * q], w[j % kRing][2 * q + 1]); };
    // The b-th block, whose first operands are in registers.  more(i): a load of the block kStages further on.
    auto work = [&](int b, auto more) __attribute__((always_inline)) {
        constexpr int kLag = 2; // a block's sum of one tile is scaled and added beside the products of the tiles after it
        float4_t part[kLag + 1];
        auto add1 = [&](int t, int e) __attribute__((always_inline)) { acc[t % kMT][t / kMT][e] = fmaf(part[t % (kLag + 1)][e], scale[t % kMT], acc[t % kMT][t / kMT][e]); };
        auto add = [&](int t) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < 4; e++) add1(t, e);
        };
#pragma unroll
        for (int i = 0; i < kMT; i++) scale[i] = sx_next[i] * sw_next;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < kTiles; t++) {
            const int i = t % kMT, j = t / kMT;
            const float4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
            if (t == kMeet) meet(kOnTheWay);
            if (i == 0) frag(frag_w, (j + kAhead) % kNT, j + kAhead < kNT ? b : b + 1, w[(j + kAhead) % kRing]);
            if constexpr (kExact) {
                float4_t s = zero;
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    s = __builtin_amdgcn_mfma_f32_16x16x32_f16(ws[j % 2][q], xs[i][q], s, 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                    if (t >= kLag) add1(t - kLag, q);
                    if (j == 0 && i + 1 < kMT) row_f16(i + 1, q);
                    if ((i * 4 + q) % kMT == 0) column_f16(j + 1, (i * 4 + q) / kMT);
                    if (t == kTiles - 1) row_f16(0, q); // (the next block's)
                    __builtin_amdgcn_sched_barrier(0);
                }
                part[t % (kLag + 1)] = s;
            } else {
                part[t % (kLag + 1)] =
                    __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_bit_cast(int8_t_, w[j % kRing]), __builtin_bit_cast(int8_t_, x[i]), zero, 0, 0, 0, 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0); // (the next product has to be on its way before the sums that wait for the one before)
            if (!kExact && t >= kLag) add(t - kLag);
            if (t >= kMeet) {
                constexpr int kLeft = kTiles - kMeet;
#pragma unroll
                for (int l = (t - kMeet) * (kLoads + kExtra) / kLeft; l < (t - kMeet + 1) * (kLoads + kExtra) / kLeft; l++) more(l);
                if (t == kMeet) read_scales(b + 1);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (j == kNT - 1) {
                frag(frag_x, i, b + 1, x[i]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int t = kTiles - kLag; t < kTiles; t++) add(t);
    };
    if constexpr (kSpans) {
        take_span(0);
        put_span(0);
    }
#pragma unroll
    for (int t = 0; t < kStages; t++) fetch(t); // (a piece has one block at least)
    meet(std::integral_constant<int, (kStages - 1) * (kLoads + kExtra)>{});
    read_scales(0);
#pragma unroll
    for (int i = 0; i < kMT; i++) frag(frag_x, i, 0, x[i]);
#pragma unroll
    for (int j = 0; j < kAhead; j++) frag(frag_w, j, 0, w[j]);
    if constexpr (kExact) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            row_f16(0, q);
            column_f16(0, q);
        }
    }
    if (count == 1) { // no whole block may be left to be loaded again: zeros then
#pragma unroll
        for (int i = 0; i < kLoads; i++) from[i] = 0;
        x0 = w0 = reinterpret_cast<const uint8_t *>(&f8_zeros);
    }
    for (int t = 0; t < count; t++) {
        if constexpr (kSpans) {
            if (t % kSpan == 0) take_span(t / kSpan + 1);
            if (t % kSpan == kSpan / 2) put_span(t / kSpan + 1);
        }
        const int b = count > 1 ? block_at(min(t + kStages, count - 1)) : 0; // (a whole one)
        work(t, [&](int i) __attribute__((always_inline)) { fetch1(b, t + kStages, i); });
    }
    wait_vmcnt<0>(); // nothing is on its way to LDS when the workgroup ends
#pragma unroll
    for (int i = 0; i < kMT; i++) {
        const int r = m0 + (wm * kMT + i) * 16 + c;
        if (r >= p.m) continue;
#pragma unroll
        for (int j = 0; j < kNT; j++) {
            const int n = nw + j * 16 + h * 4;
            if (n >= p.n) continue;
            if (pp.parts) store_row4(pp.parts + ((size_t)piece * p.m + r) * p.n, n, p.n - n, acc[i][j]);
            else store_row4(reinterpret_cast<Y *>(p.y) + (size_t)r * p.n, n, p.n - n, acc[i][j]);
        }
    }
}

// adds up the pieces in their order
template <typename Y>
__global__ __launch_bounds__(256) void matmul_f8_join_kernel(Y *y, const float *parts, int pieces, size_t count) {
    for (size_t i = (blockIdx.x * (size_t)256 + threadIdx.x) * 4; i < count; i += (size_t)gridDim.x * 1024) {
        typedef float any __attribute__((ext_vector_type(4), aligned(4)));
        if (i + 4 <= count) {
            float4_t v = *reinterpret_cast<const any *>(parts + i);
            for (int s = 1; s < pieces; s++) v += *reinterpret_cast<const any *>(parts + s * count + i);
            store_row4(y + i, 0, 4, v);
        } else {
            for (size_t e = i; e < count && e < i + 4; e++) {
                float v = parts[e];
                for (int s = 1; s < pieces; s++) v += parts[s * count + e];
                y[e] = (Y)v;
            }
        }
    }
}

// ---- which kernel ----------------------------------------------------------------------------------------------------------------------
constexpr int kFewRows = 16;
constexpr int kConvertRows = 8; // up to which rows of f16 and f32 are converted on the way (8 rows of 4096 columns 8.4 us either way, 4 6.3 / 7.7, 16 of 32000 35.7 / 31)

bool matmul_f8_converts(int m, int k) { return m <= kConvertRows && rows_f8_lds(m, k) <= kRfLds; }

// by the f16 instruction, of more rows than a few
static bool exact_products(const MatmulF8Params &p) { return !p.y_f16 || p.exact; }

// Tiles, and pieces of K.  A call takes about 5 us, tb for every block of K in every round of workgroups over the compute units, and where K is cut 3 us more and the sums' way to memory
// and back, 8 bytes per sum and piece at 4.5 bytes per ps.  (tb of the 8-bit instruction and of the f16 one, measured in products of 32 to 2048 rows.  Of the smallest tile two workgroups
// fit a compute unit, which take 1.7 times as long as one.)  The least sum is taken: 64 rows of 11008 x 4096 in two pieces 15.2 us (one 18.7, three 18.7), 131 of 4096 x 11008 in
// eight pieces of 160 rows 22.7 us (four of 128 23.8, five of 64 23.9), 1024 of 11008 x 4096 in large tiles 56 us (small ones 76), 1024 of 4096 x 4096 in small ones 27 (52).
// Over the fastest tile and number of pieces it costs 5.7 % on average with the 8-bit instruction and 1.4 % with the f16 one over 16 products each, 25 % at worst (865 x 333 x 10304).
struct TilesPlan {
    int bm, bn, tiles_m, tiles_n, pieces;
};
static TilesPlan plan_tiles(const MatmulF8Params &p, int compute_units) {
    struct Kind {
        int bm, bn;
        double tb;
    };
    const bool quick = !exact_products(p);
    const Kind kinds[] = {{64, 128, quick ? 0.43 : 0.68}, {128, 128, quick ? 0.68 : 1.15}, {160, 128, quick ? 0.66 : 1.2}, {256, quick ? 256 : 128, quick ? 1.6 : 1.76}};
    const int across = f8_blocks(p.k);
    TilesPlan best{};
    double least = 0.0;
    for (const Kind &kind : kinds) {
        TilesPlan t{kind.bm, kind.bn, (p.m + kind.bm - 1) / kind.bm, (int)(((int64_t)p.n + kind.bn - 1) / kind.bn), 1};
        const int64_t tiles = (int64_t)t.tiles_m * t.tiles_n;
        for (t.pieces = 1; t.pieces <= 16 && t.pieces * 2 <= std::max(2, across); t.pieces++) {
            const int64_t rounds = (tiles * t.pieces + compute_units - 1) / compute_units;
            const double load = kind.bm == 64 && rounds > 1 ? 0.85 * (double)rounds : (double)rounds;
            const double us = load * ((across + t.pieces - 1) / t.pieces) * kind.tb + (t.pieces > 1 ? 3.0 + (double)t.pieces * p.m * p.n * 8 / 4.5e6 : 0.0);
            if (best.bm == 0 || us < least) {
                least = us;
                best = t;
            }
        }
    }
    return best;
}

size_t matmul_f8_work_floats(const MatmulF8Params &p, int compute_units) {
    if (p.m <= kFewRows) return 0;
    const TilesPlan t = plan_tiles(p, compute_units);
    return t.pieces > 1 ? (size_t)t.pieces * p.m * p.n : 0;
}

template <int kNF, typename Y>
static hipError_t launch_rows(const RowsF8Params &p, int source, hipStream_t s) {
    const dim3 grid((unsigned)((p.p.n + 16 * kNF - 1) / (16 * kNF))), block(kRfWaves * kWave);
    if (source == kF8Codes) {
        hipLaunchKernelGGL((matmul_f8_rows_kernel<kNF, kF8Codes, Y>), grid, block, 0, s, p);
        return hipGetLastError();
    }
    const unsigned lds = (unsigned)rows_f8_lds(p.p.m, p.p.k);
    const auto kernel = source == kF8FromF16 ? matmul_f8_rows_kernel<kNF, kF8FromF16, Y> : matmul_f8_rows_kernel<kNF, kF8FromF32, Y>;
    if (lds > 24 * 1024) { // with the sums more than the 64 KiB that a kernel may have unasked
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kRfLds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kernel, grid, block, lds, s, p);
    return hipGetLastError();
}

template <int kWM, int kWN, int kMT, int kNT, int kStages, bool kExact, typename Y>
static void launch_tiles(const TilesF8Params &q, hipStream_t s) {
    const dim3 grid((unsigned)((q.tiles_m * q.tiles_n + 7) / 8 * 8), (unsigned)q.pieces);
    hipLaunchKernelGGL((matmul_f8_tiles_kernel<kWM, kWN, kMT, kNT, kStages, kExact, Y>), grid, dim3(kWM * kWN * kWave), 0, s, q);
}

template <bool kExact, typename Y>
static void launch_plan(const TilesPlan &t, const TilesF8Params &q, hipStream_t s) {
    if (t.bm == 64) launch_tiles<2, 2, 2, 4, 3, kExact, Y>(q, s);
    else if (t.bm == 128) launch_tiles<4, 2, 2, 4, 4, kExact, Y>(q, s);
    else if (t.bm == 160) launch_tiles<2, 2, 5, 4, 4, kExact, Y>(q, s);
    else launch_tiles<4, 2, 4, kExact ? 4 : 8, 2, kExact, Y>(q, s);
}

template <typename Y>
static hipError_t launch_y(const MatmulF8Params &p, const void *src, int source, int compute_units, float *ws, hipStream_t s) {
    if (p.m <= kFewRows) {
        // Columns of a workgroup: as few as give every compute unit the same share of them.  Its rows have to come in as well, so the share counts 16 kNF columns and m rows in every
        // round (us, 16 / 32 / 64 columns: one row of 4096 5.5 / 6.5 / 10.1, of 11008 9.6 / 11.2 / 10.2, of 32000 25.2 / 24.0 / 24.2; 16 rows of 32000 39 / 30.4 / 26.8).
        const RowsF8Params r{p, src};
        const int64_t tiles = ((int64_t)p.n + 15) / 16;
        auto share = [&](int nf) { return (tiles + (int64_t)nf * compute_units - 1) / ((int64_t)nf * compute_units) * (16 * nf + p.m); };
        if (share(1) <= share(2) && share(1) <= share(4)) return launch_rows<1, Y>(r, source, s);
        return share(2) <= share(4) ? launch_rows<2, Y>(r, source, s) : launch_rows<4, Y>(r, source, s);
    }
    const TilesPlan t = plan_tiles(p, compute_units);
    const TilesF8Params q{p, t.pieces > 1 ? ws : nullptr, t.pieces, t.tiles_m, t.tiles_n};
    if constexpr (sizeof(Y) == 2) {
        if (exact_products(p)) launch_plan<true, Y>(t, q, s);
        else launch_plan<false, Y>(t, q, s);
    } else {
        launch_plan<true, Y>(t, q, s);
    }
    if (t.pieces > 1) {
        const size_t count = (size_t)p.m * p.n;
        hipLaunchKernelGGL(matmul_f8_join_kernel<Y>, dim3((unsigned)std::min<size_t>((count + 1023) / 1024, 8192)), dim3(256), 0, s, (Y *)p.y, ws, t.pieces, count);
    }
    return hipGetLastError();
}

hipError_t launch_matmul_f8(const MatmulF8Params &p, const void *src, int src_f16, int compute_units, float *ws, hipStream_t s) {
    const int source = !src ? kF8Codes : src_f16 ? kF8FromF16 : kF8FromF32;
    return p.y_f16 ? launch_y<half_t>(p, src, source, compute_units, ws, s) : launch_y<float>(p, src, source, compute_units, ws, s);
}

} // namespace rlh
