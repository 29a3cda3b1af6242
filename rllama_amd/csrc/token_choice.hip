// token_choice.hip -- probabilities of rows of logits and the verification of drafted tokens against them.
#include "kernels.h"
#include "longctx.h"

namespace rlh {

typedef float float4_any __attribute__((ext_vector_type(4), aligned(4)));     // rows of any length: only the element's own alignment
typedef half_t half4_any __attribute__((ext_vector_type(4), aligned(2)));

// ---- softmax of rows ---------------------------------------------------------------------------------------------------------
// p_i = exp((x_i - m) / T) / sum_j exp((x_j - m) / T), m the row's largest.  Bound by memory.  One workgroup per row; a row of up to 32768 elements is
// read once and stays in registers (32 per thread) between the two reductions, a longer one is read three times: maximum, sum, result.
// T = 0: 1 at the first of the largest.
// Measured, rows of 32000: 320 in f16, 61 MB, 13.0 us, 4.7 TB/s; 5 in f32 5.9 us, two reductions over 1024 threads.  Rows of 128256, f16: 320, 246 MB if each is
// read and written once, 67 us, 3.7 TB/s.
template <typename T>
__device__ __forceinline__ float4_t load4(const T *x, int i, int n, float fill) {
    float4_t v;
    if (i <= n - 4) { // (i + 4 may pass 32 bits)
        if constexpr (sizeof(T) == 2) {
            const half4_any h = *reinterpret_cast<const half4_any *>(x + i);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = (float)h[j];
        } else {
            const float4_any f = *reinterpret_cast<const float4_any *>(x + i);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = f[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = i + j < n ? (float)x[i + j] : fill;
    }
    return v;
}
__device__ __forceinline__ void store4(float *y, int i, int n, float4_t v) {
    if (i <= n - 4) { // (i + 4 may pass 32 bits)
        float4_any f;
#pragma unroll
        for (int j = 0; j < 4; j++) f[j] = v[j];
        *reinterpret_cast<float4_any *>(y + i) = f;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i + j < n) y[i + j] = v[j];
    }
}

// kKeep: pieces of 4 elements that a thread keeps; 0: rows of any length, read twice.
template <typename T, int kThreads, int kKeep, bool kHot>
__global__ __launch_bounds__(kThreads) void softmax_rows_kernel(float *probs, const T *logits, int vocab, float c2 /* log2(e) / T */) {
    __shared__ float scratch_m[16], scratch_s[16];
    __shared__ int first;
    const T *x = logits + (size_t)blockIdx.x * vocab;
    float *y = probs + (size_t)blockIdx.x * vocab;
    constexpr int kStep = kThreads * 4;
    float4_t kept[kKeep > 0 ? kKeep : 1];
    // f(piece's first element, its values) over the thread's pieces
    auto pieces = [&](auto f) {
        if constexpr (kKeep > 0) {
#pragma unroll
            for (int k = 0; k < kKeep; k++) f(k * kStep + (int)threadIdx.x * 4, kept[k]);
        } else {
            for (int64_t i = threadIdx.x * 4; i < vocab; i += kStep) {
                float4_t v = load4(x, (int)i, vocab, -INFINITY);
                f((int)i, v);
            }
        }
    };
    if constexpr (kKeep > 0) {
#pragma unroll
        for (int k = 0; k < kKeep; k++) kept[k] = load4(x, k * kStep + (int)threadIdx.x * 4, vocab, -INFINITY);
    }
    if (kHot && threadIdx.x == 0) first = vocab;
    float m = -INFINITY, odd = 0.0f; // odd: NaN if a value is NaN or +infinity
    pieces([&](int, const float4_t &v) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            m = fmaxf(m, v[j]);
            if (kHot) odd += v[j] < INFINITY ? 0.0f : NAN;
        }
    });
    m = block_max(m, scratch_m);
    if constexpr (kHot) {
        odd = block_sum(odd, scratch_s);
        int mine = vocab;
        pieces([&](int i, const float4_t &v) {
#pragma unroll
            for (int j = 3; j >= 0; j--)
                if (v[j] == m && m > -INFINITY && i + j < mine) mine = i + j;
        });
        if (mine < vocab) atomicMin(&first, mine);
        __syncthreads();
        pieces([&](int i, const float4_t &) {
            float4_t p;
#pragma unroll
            for (int j = 0; j < 4; j++) p[j] = (i + j == first ? 1.0f : 0.0f) + odd;
            store4(y, i, vocab, p);
        });
        return;
    }
    const float base = m > -INFINITY ? m : 0.0f; // a row of nothing but -infinity: zeros
    // 2^20 times the exponential: the instruction flushes results below the smallest normal number, the probabilities themselves may lie there
    auto weight = [&](float v) { return __builtin_amdgcn_exp2f(fmaf(v - base, c2, 20.0f)); };
    float sum = 0.0f;
    pieces([&](int, float4_t &v) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float e = weight(v[j]);
            if (kKeep > 0) v[j] = e;
            sum += e;
        }
    });
    sum = block_sum(sum, scratch_s);
    const float r = sum == 0.0f ? 0.0f : 1.0f / sum;
    pieces([&](int i, const float4_t &v) {
        float4_t p;
#pragma unroll
        for (int j = 0; j < 4; j++) p[j] = (kKeep > 0 ? v[j] : weight(v[j])) * r;
        store4(y, i, vocab, p);
    });
}

template <typename T, bool kHot>
static void launch_softmax_t(float *probs, const T *logits, int rows, int vocab, float c2, hipStream_t s) {
    const dim3 grid((unsigned)rows);
    if (vocab <= 2048) hipLaunchKernelGGL((softmax_rows_kernel<T, 256, 2, kHot>), grid, dim3(256), 0, s, probs, logits, vocab, c2);
    else if (vocab <= 8192) hipLaunchKernelGGL((softmax_rows_kernel<T, 1024, 2, kHot>), grid, dim3(1024), 0, s, probs, logits, vocab, c2);
    else if (vocab <= 32768) hipLaunchKernelGGL((softmax_rows_kernel<T, 1024, 8, kHot>), grid, dim3(1024), 0, s, probs, logits, vocab, c2);
    else hipLaunchKernelGGL((softmax_rows_kernel<T, 1024, 0, kHot>), grid, dim3(1024), 0, s, probs, logits, vocab, c2);
}

hipError_t launch_softmax_rows(float *probs, const void *logits, int logits_f16, int rows, int vocab, float temperature, hipStream_t s) {
    const float c2 = 1.44269504088896340736f / temperature;
    const bool hot = !(c2 <= 3.4e38f); // 0, or so small that the reciprocal overflows
    if (logits_f16) {
        if (hot) launch_softmax_t<half_t, true>(probs, (const half_t *)logits, rows, vocab, c2, s);
        else launch_softmax_t<half_t, false>(probs, (const half_t *)logits, rows, vocab, c2, s);
    } else {
        if (hot) launch_softmax_t<float, true>(probs, (const float *)logits, rows, vocab, c2, s);
        else launch_softmax_t<float, false>(probs, (const float *)logits, rows, vocab, c2, s);
    }
    return hipGetLastError();
}

// ---- verification of drafted tokens ------------------------------------------------------------------------------------------
// One workgroup per sequence.  The accepted prefix needs 2 k single probabilities; the draw needs one row of p and of q.  The running sum
// is taken in whole numbers (2^-31 of a probability: one conversion per entry, 64-bit sums), so it is exact and the drawn token does
// not depend on how the row is shared: every wavefront sums a contiguous piece of the row in chunks of 256 entries (four neighbouring ones per lane), keeps
// the chunks' sums in LDS, and the wavefront whose piece holds the drawn place reads that one chunk again.
// Bound by latency: three dependent trips to memory (the ids, their probabilities, the row).  Rows of 32000: one sequence of 4 drafted tokens 9.8 us, 64 of 7
// 11.4 us (16 MB).
constexpr int kVdThreads = 1024;
constexpr int kVdWaves = kVdThreads / kWave;
constexpr int kVdChunks = 64; // per wavefront at most; longer rows have larger chunks

template <int kCtrl, int kRowMask = 0xf>
__device__ __forceinline__ uint32_t dpp_add_u32(uint32_t v) {
    return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, kRowMask, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_sum_u32(uint32_t v) { // wave-uniform
    v = dpp_add_u32<kDppQuadPerm1032>(v);
    v = dpp_add_u32<kDppQuadPerm2301>(v);
    v = dpp_add_u32<kDppRowHalfMirror>(v);
    v = dpp_add_u32<kDppRowMirror>(v);
    v = dpp_add_u32<kDppRowBcast15, 0xa>(v);
    v = dpp_add_u32<kDppRowBcast31, 0xc>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

__global__ __launch_bounds__(kVdThreads) void verify_draft_kernel(VerifyParams p) {
    __shared__ int sh_count, sh_sub, sh_pick;
    __shared__ uint64_t piece_sum[kVdWaves], chunk_sum[kVdWaves][kVdChunks];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
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
    const int per_wave = (int)((((int64_t)V + kVdWaves - 1) / kVdWaves + 255) / 256); // in groups of 256
    const int chunk = (per_wave + kVdChunks - 1) / kVdChunks * 256, chunks = (per_wave * 256 + chunk - 1) / chunk;
    const int64_t lo = (int64_t)wave * chunks * chunk; // (may lie past the row)
    const float mf = fminf(fmaxf(u[k] * 16777216.0f, 0.0f), 16777215.0f); // (NaN: 0)
    const uint64_t m = (uint64_t)mf;

    for (int pass = 0; pass < 2; pass++) { // the second one only where nothing is left of max(p - q, 0): p itself
        typedef __attribute__((ext_vector_type(4))) uint32_t weights_t;
        auto weights = [&](int64_t at) -> weights_t { // of entries at .. at + 3
            weights_t w = {0u, 0u, 0u, 0u};
            if (at >= V) return w;
            float4_t v = load4(prow, (int)at, V, 0.0f);
            if (pass == 0 && qrow) v -= load4(qrow, (int)at, V, 0.0f);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (pass == 0 && at + j == certain) v[j] -= 1.0f;
                w[j] = (uint32_t)rintf(fminf(fmaxf(v[j], 0.0f), 1.0f) * 2147483648.0f);
            }
            return w;
        };
        // sum over the lanes of up to four weights each: halves of 16 bits apart, so that 32-bit sums hold them
        auto lanes_sum = [&](const weights_t &w) -> uint64_t {
            uint32_t a = 0, h = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                a += w[j] & 0xffffu;
                h += w[j] >> 16;
            }
            return (uint64_t)wave_sum_u32(a) + ((uint64_t)wave_sum_u32(h) << 16);
        };
        uint64_t sum = 0;
        for (int c = 0; c < chunks; c++) {
            uint64_t part = 0;
            for (int i = 0; i < chunk; i += 256) part += lanes_sum(weights(lo + (int64_t)c * chunk + i + lane * 4));
            if (lane == 0) chunk_sum[wave][c] = part;
            sum += part;
        }
        if (lane == 0) piece_sum[wave] = sum;
        __syncthreads();
        uint64_t total = 0, before = 0;
        for (int w = 0; w < kVdWaves; w++) {
            if (w == wave) before = total;
            total += piece_sum[w];
        }
        const uint64_t place = (total >> 24) * m + (((total & 0xffffff) * m) >> 24);
        if (total > 0) {
            if (before <= place && place < before + sum) { // this wavefront's piece holds the drawn place
                int c = 0;
                while (before + chunk_sum[wave][c] <= place) before += chunk_sum[wave][c++];
                for (int i = 0; i < chunk; i += 256) {
                    const int64_t at = lo + (int64_t)c * chunk + i + lane * 4;
                    const weights_t w = weights(at);
                    uint64_t run = (uint64_t)w[0] + w[1] + w[2] + w[3]; // up to this lane's last
#pragma unroll
                    for (int off = 1; off < kWave; off <<= 1) {
                        const uint64_t up = (uint64_t)__shfl_up((unsigned long long)run, off, kWave);
                        if (lane >= off) run += up;
                    }
                    const uint64_t found = __ballot(before + run > place);
                    if (found) {
                        if (lane == __builtin_ctzll(found)) {
                            uint64_t at_run = before + run - w[0] - w[1] - w[2] - w[3];
                            int j = 0;
                            while (j < 3 && at_run + w[j] <= place) at_run += w[j++];
                            sh_pick = (int)(at + j);
                        }
                        break;
                    }
                    before += (uint64_t)__shfl((unsigned long long)run, kWave - 1, kWave);
                }
            }
            break;
        }
        __syncthreads(); // the sums are written again
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
