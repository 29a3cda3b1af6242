// f8.h -- tensors of 8-bit floating point (RLH_F8, RLH_F8_TILES) as the kernels see them.
//
// A tensor [rows x cols], cols a multiple of 16, is one buffer: the e4m3 codes, row after row, then the scales in f32: one for every 128 columns of
// a row (activations), or one for every tile of 128 rows and 128 columns (weights).  A value is code * scale.  Behind the last column of a row whose
// length is no multiple of 128 there is nothing: its last block is shorter.
#pragma once

#include "device_utils.h"
#include "f8_layout.h"

namespace rlh {

constexpr float kF8Largest = 448.0f; // of e4m3

struct EightRef {
    uint8_t *codes;
    float *scales;
    int rows; // that share a scale: 1 or 128
};

// Scale and factor of a block whose largest value is `top` (finite): value = code * scale, code = e4m3(value * factor).  The bound keeps both normal numbers; below it
// a block is all but zero.  (The factor is a reciprocal and a product, two roundings, which is what torch makes of a number divided by a tensor: codes made so there and here are the
// same.  A division rounds once; one code in 1e5 then falls on the other side of a tie.)
struct F8Scale {
    float scale, factor;
    __device__ explicit F8Scale(float top) {
        const float a = fmaxf(top, kF8Largest * 1.1754943508222875e-38f);
        scale = a / kF8Largest;
        factor = kF8Largest * (1.0f / a);
    }
};
// codes of two values, in the low or the high half of `word`; the conversion rounds ties to even, and codes above the largest one would read as NaN
template <bool kHigh>
__device__ __forceinline__ int f8_codes(float a, float b, int word) {
    a = fminf(fmaxf(a, -kF8Largest), kF8Largest);
    b = fminf(fmaxf(b, -kF8Largest), kF8Largest);
    return __builtin_amdgcn_cvt_pk_fp8_f32(a, b, word, kHigh);
}
// the values of a word's codes 2 half, 2 half + 1 as f16 numbers, exactly
template <bool kHigh>
__device__ __forceinline__ half2_t f8_pair_f16(uint32_t word) {
    return __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)word, 1.0f, kHigh));
}

} // namespace rlh
