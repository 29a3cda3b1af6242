// gemm_f8.hip -- products of 8-bit floating point with a scale for each block of 128:
//   y[r, c] = sum_b sx[r, b] sw[c / 128, b] sum_{k in block b} x[r, k] w[c, k].
#include "kernels.h"
#include "answers.h"

namespace rlh {

// One thread per result.
template <typename T>
__global__ __launch_bounds__(256) void matmul_f8_kernel(MatmulF8Params p) {
    const int c = blockIdx.x * 16 + threadIdx.x % 16;
    const int64_t r = (int64_t)blockIdx.y * 16 + threadIdx.x / 16;
    if (r >= p.m || c >= p.n) return;
    const int across = f8_blocks(p.k);
    float y = 0.0f;
    for (int b = 0; b < across; b++) {
        float part = 0.0f;
        for (int k = b * kF8Block; k < min(p.k, (b + 1) * kF8Block); k += 16) {
            const uint4_t x = *reinterpret_cast<const uint4_t *>(p.x.codes + (size_t)r * p.k + k), w = *reinterpret_cast<const uint4_t *>(p.w.codes + (size_t)c * p.k + k);
            for (int i = 0; i < 4; i++) {
                const half2_t x0 = f8_pair_f16<false>(x[i]), x1 = f8_pair_f16<true>(x[i]), w0 = f8_pair_f16<false>(w[i]), w1 = f8_pair_f16<true>(w[i]);
                part = fmaf((float)x0[0], (float)w0[0], part);
                part = fmaf((float)x0[1], (float)w0[1], part);
                part = fmaf((float)x1[0], (float)w1[0], part);
                part = fmaf((float)x1[1], (float)w1[1], part);
            }
        }
        y = fmaf(part, p.x.scales[(size_t)r * across + b] * p.w.scales[(size_t)(c / kF8Block) * across + b], y);
    }
    reinterpret_cast<T *>(p.y)[(size_t)r * p.n + c] = (T)y;
}

hipError_t launch_matmul_f8(const MatmulF8Params &p, int compute_units, hipStream_t s) {
    const dim3 grid((unsigned)((p.n + 15) / 16), (unsigned)((p.m + 15) / 16));
    if (p.y_f16) hipLaunchKernelGGL(matmul_f8_kernel<half_t>, grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL(matmul_f8_kernel<float>, grid, dim3(256), 0, s, p);
    return hipGetLastError();
}

} // namespace rlh
