// attn_window.hip -- attention over cache planes of 16, 32 or 4 bits with a sliding window and first tokens that stay visible.
//
// The row at position p sees the positions t <= p with t < sinks or t > p - window:
//   out = sum_t w_t v_t / sum_t w_t,  w_t = exp(q . k_t / sqrt(hd) - m),  m the largest score,
// in one pass over the positions with a running (m, sum w, sum w v) per row.
//
// The rows that share a key and value head (n rows of n_heads / n_kv heads) are taken 16 at a time, so that every cached value is read
// once for all of them and both products go through the matrix cores, transposed so that a row is a column of both:
//   S^T [position x row] = K [position x dim] . q^T,     O^T [dim x row] += V^T [dim x position] . W [position x row]
// With 16 x 16 tiles lane l holds column l % 16 of a result, rows 4 (l / 16) + i: a row's maximum, sum and rescaling factor live in the
// lanes of its column, and the weights a lane has just formed are the operand it has to supply to the second product, if that product's
// inner index runs over the positions in the order 4 h + j (j < 4), 16 + 4 h + j - 4 (h = l / 16).  V then has to be read by position and
// supplied by dimension: a lane loads the hd / 16 neighbouring dims of each of its eight positions (whole rows of V by 16 lanes) and
// transposes them in registers with byte permutes, so cached rows go from memory into registers and nowhere else: no LDS, no barrier in
// the loop.  Tile e of O^T is made of the dims hd / 16 * m + e (m = 0 .. 15).
//
// Two arithmetics.  16 bits: f16 operands, v_mfma_f32_16x16x32_f16, and nothing but the result is rounded to f16.  A weight is the sum of two f16 numbers, 22 bits, and takes
// two products with V (one row behind 383 positions 7.3 -> 7.5 us, 16 texts with a window 16.2 -> 16.5, 65700 positions in 4 bits 27.4 -> 28.1; rounded to f16 the weights left
// 1.6e-4 of the result's size).  A value of 4 bits is 16 * code * (upper part of the scale / 16) + code * (rest) + lowest, two products that f16 holds exactly for every
// scale and a term that is the same for 32 dims, and each goes through the matrix cores by itself.  32 bits: everything in f32 through v_mfma_f32_16x16x4_f32; also
// taken where f16 queries meet an f32 cache, whose values f16 may not hold.
//
// A text is cut into pieces when there are few rows: every workgroup leaves its (m, sum, O) in work memory and a second launch joins them.
//
// Measured: 16 texts, one row each over a window of 1024 and 4, 32 heads on 8 of 128: 63 MB in 13.4 us, 4.7 TB/s, and 3.9 us of join.  5 rows in f32 behind 2107
// positions of 32 heads: 69 MB in 15.0 us, 4.6 TB/s.  Both are bound by memory.  One row behind 65700 positions in 4 bits, 64 heads on 8: 84 MB in 25.8 us,
// 3.3 TB/s: nothing is saturated (vector ALU 43 %, matrix cores 15 %); its 166 registers leave one workgroup to a compute unit, two wavefronts per SIMD, each of which waits for
// the loads of a step 41 % of its time.  One row behind 383 positions, 6.3 MB: 7.6 us, a chain of latencies.
#include "kernels.h"
#include "attn_rows_device.h"

#include <algorithm>

namespace rlh {

template <typename AC, typename QT, typename CT, int HD>
__global__ __launch_bounds__(kAwThreads) void attn_rows_kernel(AttnCutParams pp) {
    __shared__ RowsShared<HD> shared;
    attn_rows<AC, QT, CT, HD>(WindowView(pp), shared, blockIdx.z, blockIdx.y, blockIdx.x);
}

template <typename AC, typename QT, typename CT, int HD>
static hipError_t launch_rows(const AttnCutParams &p, hipStream_t s) {
    const int rows = p.a.n * (p.a.n_heads / p.a.n_kv);
    const dim3 grid((unsigned)p.pieces, (unsigned)((rows + kAwRows - 1) / kAwRows), (unsigned)(p.a.n_seqs * p.a.n_kv));
    hipLaunchKernelGGL((attn_rows_kernel<AC, QT, CT, HD>), grid, dim3(kAwThreads), 0, s, p);
    if (p.pieces > 1) launch_attn_join<QT, HD, kAwRows, Step<AC, CT, HD>::kPositions>(p, s);
    return hipGetLastError();
}
template <typename AC, typename QT, typename CT>
static hipError_t launch_rows_hd(const AttnCutParams &p, hipStream_t s) {
    switch (p.a.head_dim) {
    case 32: return launch_rows<AC, QT, CT, 32>(p, s);
    case 64: return launch_rows<AC, QT, CT, 64>(p, s);
    case 128: return launch_rows<AC, QT, CT, 128>(p, s);
    default: return hipErrorInvalidValue;
    }
}

// f32 arithmetic is needed for f32 queries and where an f32 cache may hold what f16 cannot
static bool f16_arithmetic(const AttnWindowParams &p) { return p.f16 && p.cache != kPlaneF32; }

// How the texts are cut: pieces of `piece_steps` steps, at most `pieces` of them; and about what the call takes.
struct RowsCut {
    int pieces, piece_steps;
    int most; // pieces of a text of any length
    double us;
};
static RowsCut cut_rows(const AttnWindowParams &p, int compute_units) {
    const int group = p.n_heads / p.n_kv, step = f16_arithmetic(p) ? 32 : 16;
    const int64_t rows = (int64_t)p.n * group, tiles = (rows + kAwRows - 1) / kAwRows, units = tiles * p.n_seqs * p.n_kv;
    // no tile has more steps than this: its rows' positions are at most `apart` from each other
    const int64_t apart = std::min<int64_t>(p.n - 1, (kAwRows - 2) / group + 1);
    int64_t steps = 1;
    double keys = 0.0; // that an average tile looks at, summed over the sequences
    for (int b = 0; b < p.n_seqs; b++) {
        const int64_t last = (int64_t)p.start[b] + p.n - 1;
        if (last < 0) continue;
        int64_t count = (last + step) / step;
        double mean = 0.5 * (double)(std::max(0, p.start[b]) + last + 1);
        if (p.window > 0) {
            count = std::min(count, (p.window - 1 + apart + step) / step) + (p.sinks + step - 1) / step;
            mean = std::min(mean, (double)p.window + apart + p.sinks);
        }
        if (last >= p.max_seq_len) count++; // the ring's end cuts a step in two
        steps = std::max(steps, count);
        keys += mean;
    }
    // About one workgroup per compute unit, with a step for each wavefront at least.  Up to two and a half steps per wavefront are not cut, nor up to four where there
    // would be two pieces: joining costs a launch, about 3 us (f16, us, whole / cut; 32 heads, one text: 384 positions 7.4 / 8.7 in two pieces, 600: 9.3 / 9.5, 768:
    // 10.5 / 9.7, 1024: 12.0 / 9.7; 16 texts of 8 key and value heads, in two pieces: 600: 9.6 / 11.3, 1000: 13.5 / 13.7).
    const int64_t want = std::max<int64_t>(1, compute_units / units);
    const int64_t n = 2 * steps <= (want == 2 ? 8 : 5) * kAwWaves ? 1 : std::min<int64_t>({want, (steps + kAwWaves - 1) / kAwWaves, kMaxPieces});
    RowsCut cut;
    cut.most = (int)std::min<int64_t>(want, kMaxPieces);
    cut.piece_steps = (int)((steps + n - 1) / n);
    cut.pieces = (int)((steps + cut.piece_steps - 1) / cut.piece_steps);
    cut.us = 5.0 + (cut.pieces > 1 ? 3.5 : 0.0) + units * 0.01 + tiles * p.n_kv * keys * p.head_dim / 128 * 30e-6 + (double)cut.piece_steps * step * p.head_dim / 128 * 4e-3;
    return cut;
}

// The tiles of attn_tiles.hip take 128 rows at once, this kernel 16: it reads K and V once per 16 rows, but has more workgroups, no second rounding of 4-bit values
// and more wavefronts per key.  Both sides' estimates were fitted to measured shapes (17 .. 2400 rows per key and value head, 0 .. 8000 positions, f16 and 4 bits);
// over 262 of them going by the estimates costs 1.5 % over always taking the faster one, 60 % at worst, a fixed limit of 64 rows 11 to 13 %, 140 at worst.  (us, this / tiles, 32 heads of 128: 128 rows from position 0
// 7.1 / 8.8, behind 500 14.9 / 20.0, behind 2000 41 / 21.7; 64 rows behind 4000 44 / 22.)
static bool tiles_take(const AttnWindowParams &p, int compute_units) {
    return f16_arithmetic(p) && !p.exact && p.n * (int64_t)(p.n_heads / p.n_kv) > kAwRows && attn_tiles_us(p, compute_units) < cut_rows(p, compute_units).us;
}

int64_t attn_window_most_rows(const AttnWindowParams &p, int compute_units) {
    if ((int64_t)p.n_seqs * p.n_kv > 65535) return 0;
    return 65535 * (int64_t)(tiles_take(p, compute_units) ? attn_tiles_rows() : kAwRows);
}

size_t attn_window_work_floats(const AttnWindowParams &p, int compute_units) {
    if (tiles_take(p, compute_units)) return attn_tiles_work_floats(p, compute_units);
    const RowsCut cut = cut_rows(p, compute_units);
    return cut.pieces > 1 ? (size_t)p.n * p.n_heads * p.n_seqs * cut.most * (p.head_dim + 2) : 0;
}

hipError_t launch_attn_window(const AttnWindowParams &a, int compute_units, float *ws, hipStream_t s) {
    if (tiles_take(a, compute_units)) return launch_attn_tiles(a, compute_units, ws, s);
    AttnCutParams p;
    p.a = a;
    p.ws = ws;
    const RowsCut cut = cut_rows(a, compute_units);
    p.pieces = cut.pieces;
    p.piece_steps = cut.piece_steps;
    switch (a.cache * 2 + a.f16) {
    case kPlaneF16 * 2: return launch_rows_hd<float, float, half_t>(p, s);
    case kPlaneF16 * 2 + 1: return launch_rows_hd<half_t, half_t, half_t>(p, s);
    case kPlaneF32 * 2: return launch_rows_hd<float, float, float>(p, s);
    case kPlaneF32 * 2 + 1: return launch_rows_hd<float, half_t, float>(p, s);
    case kPlaneQ4 * 2: return launch_rows_hd<float, float, Quant4>(p, s);
    case kPlaneQ4 * 2 + 1: return launch_rows_hd<half_t, half_t, Quant4>(p, s);
    default: return hipErrorInvalidValue;
    }
}

} // namespace rlh
