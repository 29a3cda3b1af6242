// f8_layout.h -- blocks of 8-bit tensors, and where a product of few rows keeps the rows that it converts (gemm_f8.hip).  Arithmetic on sizes alone, so it is checked on the
// CPU over all sizes.
#pragma once

#include <cstddef>

namespace rlh {

constexpr int kF8Block = 128; // columns that share a scale

constexpr int f8_blocks(int cols) { return (cols + kF8Block - 1) / kF8Block; }

// A wavefront's region of LDS: the codes [block][row] of its share of the blocks, then their scales.  Rows are padded, so that they lie in different banks, and read sixteen bytes at a
// time: every region starts at a multiple of that.  (One behind the other without it: one row of 11008 into 4096 columns 10.8 us, 10.4 so; 7 of 5120 into 5120 11.1, 10.9.)
constexpr int kRfWaves = 8;
constexpr int kRfRow = kF8Block + 16;
constexpr int rows_f8_share(int k) { return (f8_blocks(k) + kRfWaves - 1) / kRfWaves; } // blocks of a wavefront
constexpr size_t rows_f8_region(int m, int k) { return ((size_t)rows_f8_share(k) * m * (kRfRow + sizeof(float)) + 15) / 16 * 16; }
constexpr size_t rows_f8_lds(int m, int k) { return kRfWaves * rows_f8_region(m, k); }

} // namespace rlh
