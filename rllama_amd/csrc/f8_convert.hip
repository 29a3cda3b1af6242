// f8_convert.hip -- tensors of f16 and f32 to 8-bit floating point with a scale for each block, and back.  Memory bound: everything is read once and written once, a
// block's largest value found by the lanes that hold it.  16 rows of 4096 take 3 us (a launch), 2048 of 5120 in f16 6.2 (5.1 TB/s), 32768 of 8192 138 (5.8).
#include "kernels.h"
#include "answers.h"

#include <algorithm>

namespace rlh {

// Sixteen values from element `index` on, a multiple of 16 of a tensor of type T
template <typename T>
__device__ __forceinline__ void load16_values(const T *src, size_t index, float (&v)[16]) {
    const PlaneRef p{const_cast<T *>(src), nullptr};
    float a[8], b[8];
    plane_load8<T>(p, index, a);
    plane_load8<T>(p, index + 8, b);
#pragma unroll
    for (int i = 0; i < 8; i++) {
        v[i] = a[i];
        v[i + 8] = b[i];
    }
}

// A block is kRows rows of 128 columns; eight neighbouring lanes have 16 columns each of a row.  kRows = 1: a workgroup of 256 threads takes 32 blocks.  128: one.
template <typename T, int kRows>
__global__ __launch_bounds__(256) void f8_encode_kernel(EightRef dst, const T *src, int rows, int cols, int across, int64_t blocks) {
    constexpr int kPieces = kRows == 1 ? 1 : kRows * 8 / 256; // of 16 values that a thread keeps
    const int tid = threadIdx.x;
    const int64_t block = kRows == 1 ? (int64_t)blockIdx.x * 32 + tid / 8 : (int64_t)blockIdx.x;
    if (kRows == 1 && block >= blocks) return;
    const int64_t down = block / across;
    const int c = (int)(block - down * across) * kF8Block + (tid % 8) * 16;
    float v[kPieces][16], top = 0.0f, odd = 0.0f; // odd: NaN if some value is not finite
#pragma unroll
    for (int k = 0; k < kPieces; k++) {
        const int64_t r = kRows == 1 ? down : down * kRows + k * 32 + tid / 8;
        if (r < rows && c < cols) {
            load16_values(src, (size_t)r * cols + c, v[k]);
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) v[k][i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
            top = fmaxf(top, fabsf(v[k][i]));
            odd += v[k][i] - v[k][i];
        }
    }
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) {
        top = fmaxf(top, __shfl_xor(top, off, kWave));
        odd += __shfl_xor(odd, off, kWave);
    }
    if constexpr (kRows > 1) {
        __shared__ float scratch[16], scratch2[16];
        top = block_max(top, scratch);
        odd = block_sum(odd, scratch2);
    }
    const F8Scale by(top);
#pragma unroll
    for (int k = 0; k < kPieces; k++) {
        const int64_t r = kRows == 1 ? down : down * kRows + k * 32 + tid / 8;
        if (r >= rows || c >= cols) continue;
        uint4_t w;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            int x = f8_codes<false>(v[k][4 * i] * by.factor, v[k][4 * i + 1] * by.factor, 0);
            x = f8_codes<true>(v[k][4 * i + 2] * by.factor, v[k][4 * i + 3] * by.factor, x);
            w[i] = odd == 0.0f ? (uint32_t)x : 0u;
        }
        *reinterpret_cast<uint4_t *>(dst.codes + (size_t)r * cols + c) = w;
    }
    if (kRows == 1 ? tid % 8 == 0 : tid == 0) dst.scales[block] = odd == 0.0f ? by.scale : NAN;
}

template <typename T>
__global__ __launch_bounds__(256) void f8_decode_kernel(T *dst, EightRef src, int cols, int across, size_t pieces) {
    for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < pieces; i += (size_t)gridDim.x * 256) {
        const size_t r = i / (cols / 16);
        const int c = (int)(i - r * (cols / 16)) * 16;
        const float scale = src.scales[(r / src.rows) * across + c / kF8Block];
        const uint4_t w = *reinterpret_cast<const uint4_t *>(src.codes + i * 16);
#pragma unroll
        for (int k = 0; k < 2; k++) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const half2_t a = f8_pair_f16<false>(w[2 * k + j]), b = f8_pair_f16<true>(w[2 * k + j]);
                v[4 * j] = (float)a[0] * scale;
                v[4 * j + 1] = (float)a[1] * scale;
                v[4 * j + 2] = (float)b[0] * scale;
                v[4 * j + 3] = (float)b[1] * scale;
            }
            plane_store8<T>(PlaneRef{dst, nullptr}, i * 16 + 8 * k, v);
        }
    }
}

template <typename T>
static void launch_encode(const EightRef &dst, const T *src, int rows, int cols, hipStream_t s) {
    const int across = f8_blocks(cols);
    if (dst.rows == 1) {
        const int64_t step = std::max<int64_t>(1, (1 << 28) / across); // rows of a launch, which takes less than 2^32 threads
        for (int64_t r0 = 0; r0 < rows; r0 += step) {
            const int part = (int)std::min<int64_t>(step, rows - r0);
            const int64_t blocks = (int64_t)part * across;
            hipLaunchKernelGGL((f8_encode_kernel<T, 1>), dim3((unsigned)((blocks + 31) / 32)), dim3(256), 0, s, EightRef{dst.codes + (size_t)r0 * cols, dst.scales + (size_t)r0 * across, 1},
                               src + (size_t)r0 * cols, part, cols, across, blocks);
        }
    } else {
        const int64_t blocks = (int64_t)f8_blocks(rows) * across;
        hipLaunchKernelGGL((f8_encode_kernel<T, kF8Block>), dim3((unsigned)blocks), dim3(256), 0, s, dst, src, rows, cols, across, blocks);
    }
}

hipError_t launch_f8_encode(const EightRef &dst, const void *src, int src_f16, int rows, int cols, hipStream_t s) {
    if (src_f16) launch_encode(dst, (const half_t *)src, rows, cols, s);
    else launch_encode(dst, (const float *)src, rows, cols, s);
    return hipGetLastError();
}

hipError_t launch_f8_decode(void *dst, int dst_f16, const EightRef &src, int rows, int cols, hipStream_t s) {
    const size_t pieces = (size_t)rows * (cols / 16);
    const dim3 grid((unsigned)std::min<size_t>((pieces + 255) / 256, 8192));
    if (dst_f16) hipLaunchKernelGGL(f8_decode_kernel<half_t>, grid, dim3(256), 0, s, (half_t *)dst, src, cols, f8_blocks(cols), pieces);
    else hipLaunchKernelGGL(f8_decode_kernel<float>, grid, dim3(256), 0, s, (float *)dst, src, cols, f8_blocks(cols), pieces);
    return hipGetLastError();
}

} // namespace rlh
