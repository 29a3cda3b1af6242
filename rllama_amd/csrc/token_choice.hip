// token_choice.hip -- probabilities of rows of logits and the verification of drafted tokens against them.
#include "kernels.h"
#include "longctx.h"

namespace rlh {

// ---- softmax of rows ---------------------------------------------------------------------------------------------------------
// p_i = exp((x_i - m) / T) / sum_j exp((x_j - m) / T), m the row's largest.  Bound by memory: a row is read once for m and the running
// sum and once more (from the caches) to be written.
constexpr int kSmThreads = 1024;

// sums and maxima over the block; `scratch` has a float per wavefront and is free again on return
__device__ __forceinline__ float all_max(float v, float *scratch) {
    v = block_max(v, scratch);
    __syncthreads();
    return v;
}
__device__ __forceinline__ float all_sum(float v, float *scratch) {
    v = block_sum(v, scratch);
    __syncthreads();
    return v;
}

template <typename T>
__global__ __launch_bounds__(kSmThreads) void softmax_rows_kernel(float *probs, const T *logits, int vocab, float inv_t) {
    __shared__ float scratch[16];
    const T *x = logits + (size_t)blockIdx.x * vocab;
    float *y = probs + (size_t)blockIdx.x * vocab;
    float m = -INFINITY, odd = 0.0f;
    for (int i = threadIdx.x; i < vocab; i += kSmThreads) {
        const float v = (float)x[i];
        m = fmaxf(m, v);
        if (v != v) odd = v;
    }
    m = all_max(m, scratch);
    float sum = odd;
    for (int i = threadIdx.x; i < vocab; i += kSmThreads) sum += m > -INFINITY ? expf(((float)x[i] - m) * inv_t) : 0.0f;
    sum = all_sum(sum, scratch);
    const float r = 1.0f / sum;
    for (int i = threadIdx.x; i < vocab; i += kSmThreads) y[i] = sum == 0.0f ? 0.0f : expf(((float)x[i] - m) * inv_t) * r;
}

// temperature 0: 1 at the first of the largest
template <typename T>
__global__ __launch_bounds__(kSmThreads) void one_hot_rows_kernel(float *probs, const T *logits, int vocab) {
    __shared__ float scratch[16];
    __shared__ int first;
    const T *x = logits + (size_t)blockIdx.x * vocab;
    float *y = probs + (size_t)blockIdx.x * vocab;
    float m = -INFINITY, odd = 0.0f;
    for (int i = threadIdx.x; i < vocab; i += kSmThreads) {
        const float v = (float)x[i];
        m = fmaxf(m, v);
        odd += v < INFINITY ? 0.0f : NAN; // NaN and +infinity
    }
    if (threadIdx.x == 0) first = vocab;
    m = all_max(m, scratch);
    odd = all_sum(odd, scratch);
    for (int i = threadIdx.x; i < vocab; i += kSmThreads) {
        if ((float)x[i] == m && m > -INFINITY) {
            atomicMin(&first, i);
            break;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < vocab; i += kSmThreads) y[i] = (i == first ? 1.0f : 0.0f) + odd;
}

hipError_t launch_softmax_rows(float *probs, const void *logits, int logits_f16, int rows, int vocab, float temperature, hipStream_t s) {
    const dim3 grid((unsigned)rows), block(kSmThreads);
    const float inv_t = 1.0f / temperature;
    if (!(inv_t <= 3.4e38f)) { // 0, or so small that the reciprocal overflows
        if (logits_f16) hipLaunchKernelGGL(one_hot_rows_kernel<half_t>, grid, block, 0, s, probs, (const half_t *)logits, vocab);
        else hipLaunchKernelGGL(one_hot_rows_kernel<float>, grid, block, 0, s, probs, (const float *)logits, vocab);
    } else if (logits_f16) hipLaunchKernelGGL(softmax_rows_kernel<half_t>, grid, block, 0, s, probs, (const half_t *)logits, vocab, inv_t);
    else hipLaunchKernelGGL(softmax_rows_kernel<float>, grid, block, 0, s, probs, (const float *)logits, vocab, inv_t);
    return hipGetLastError();
}

// ---- verification of drafted tokens ------------------------------------------------------------------------------------------
// One workgroup per sequence.  The accepted prefix needs 2 k single probabilities; the draw needs one row of p and of q.  The running sum
// is taken in whole numbers (2^-31 of a probability: one conversion per entry, 64-bit sums), so it is exact and the drawn token does
// not depend on how the row is shared between threads: every wavefront sums a contiguous piece of the row, then the piece that holds the
// drawn place is searched.
constexpr int kVdThreads = 1024;
constexpr int kVdWaves = kVdThreads / kWave;

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += (uint64_t)__shfl_xor((unsigned long long)v, off, kWave);
    return v;
}

__global__ __launch_bounds__(kVdThreads) void verify_draft_kernel(VerifyParams p) {
    __shared__ int sh_count, sh_sub, sh_pick;
    __shared__ uint64_t piece_sum[kVdWaves];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int b = blockIdx.x, k = p.k, V = p.vocab;
    const int32_t *ids = p.drafted + (size_t)b * k;
    const float *u = p.uniforms + (size_t)b * (k + 1);
    int32_t *out = p.out + (size_t)b * (k + 2);

    // the first drafted token that is not accepted; whether the draft's own row is taken off there
    if (wave == 0) {
        int count = k, sub = 0;
        for (int base = 0; base < k && count == k; base += kWave) {
            const int i = base + lane;
            bool stop = false, inside = false;
            if (i < k) {
                const int id = ids[i];
                inside = id >= 0 && id < V;
                stop = true;
                if (inside) {
                    const float q = p.draft ? p.draft[((size_t)b * k + i) * V + id] : 1.0f;
                    stop = !(u[i] * q < p.target[((size_t)b * (k + 1) + i) * V + id]);
                }
            }
            const uint64_t stops = __ballot(stop);
            if (stops) {
                const int at = __builtin_ctzll(stops);
                count = base + at;
                sub = __shfl(inside ? 1 : 0, at, kWave);
            }
        }
        if (lane == 0) {
            sh_count = count;
            sh_sub = sub;
            sh_pick = V;
        }
    }
    __syncthreads();
    const int count = sh_count;
    const float *prow = p.target + ((size_t)b * (k + 1) + count) * V;
    const float *qrow = sh_sub && p.draft ? p.draft + ((size_t)b * k + count) * V : nullptr;
    const int certain = sh_sub && !p.draft ? ids[count] : -1; // a draft without probabilities: all of it on the token itself
    const int piece = (V + kVdWaves - 1) / kVdWaves, lo = min(V, wave * piece), hi = min(V, lo + piece);
    const float mf = fminf(fmaxf(u[k] * 16777216.0f, 0.0f), 16777215.0f); // (NaN: 0)
    const uint64_t m = (uint64_t)mf;

    for (int pass = 0; pass < 2; pass++) { // the second one only where nothing is left of max(p - q, 0): p itself
        auto weight = [&](int i) -> uint64_t {
            float w = prow[i];
            if (pass == 0) {
                if (qrow) w -= qrow[i];
                if (i == certain) w = w - 1.0f;
            }
            return (uint32_t)rintf(fminf(fmaxf(w, 0.0f), 1.0f) * 2147483648.0f);
        };
        uint64_t sum = 0;
        for (int i = lo + lane; i < hi; i += kWave) sum += weight(i);
        sum = wave_sum_u64(sum);
        if (lane == 0) piece_sum[wave] = sum;
        __syncthreads();
        uint64_t total = 0;
        for (int w = 0; w < kVdWaves; w++) total += piece_sum[w];
        const uint64_t place = (total >> 24) * m + (((total & 0xffffff) * m) >> 24);
        if (total > 0) {
            uint64_t before = 0;
            for (int w = 0; w < wave; w++) before += piece_sum[w];
            if (before <= place && place < before + sum) { // this wavefront's piece holds the drawn place
                for (int base = lo; base < hi; base += kWave) {
                    const int i = base + lane;
                    uint64_t run = i < hi ? weight(i) : 0;
#pragma unroll
                    for (int off = 1; off < kWave; off <<= 1) {
                        const uint64_t up = (uint64_t)__shfl_up((unsigned long long)run, off, kWave);
                        if (lane >= off) run += up;
                    }
                    const uint64_t found = __ballot(before + run > place);
                    if (found) {
                        if (lane == 0) sh_pick = base + __builtin_ctzll(found);
                        break;
                    }
                    before += (uint64_t)__shfl((unsigned long long)run, kWave - 1, kWave);
                }
            }
            break;
        }
        __syncthreads(); // piece_sum is written again
    }
    __syncthreads();
    const int pick = sh_pick < V ? sh_pick : -1;
    if (tid == 0) out[0] = count;
    for (int i = tid; i <= k; i += kVdThreads) out[1 + i] = i < count ? ids[i] : i == count ? pick : -1;
}

hipError_t launch_verify_draft(const VerifyParams &p, hipStream_t s) {
    hipLaunchKernelGGL(verify_draft_kernel, dim3((unsigned)p.n_seqs), dim3(kVdThreads), 0, s, p);
    return hipGetLastError();
}

} // namespace rlh
