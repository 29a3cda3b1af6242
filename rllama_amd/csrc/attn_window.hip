// attn_window.hip -- attention over cache planes of 16, 32 or 4 bits with a sliding window and first tokens that stay visible.
//
// The row at position p sees the positions t <= p with t < sinks or t > p - window:
//   out = sum_t w_t v_t / sum_t w_t,  w_t = exp(q . k_t / sqrt(hd) - m),  m the largest score.
// One pass with a running (m, sum w, sum w v).  One workgroup per row and head; hd / 8 lanes hold one position, 8 elements each.
#include "kernels.h"
#include "longctx.h"

namespace rlh {

constexpr int kAwThreads = 256;

template <typename QT, typename CT, int HD>
__global__ __launch_bounds__(kAwThreads) void attn_window_kernel(AttnWindowParams p) {
    constexpr int kLanes = HD / 8;
    constexpr int kSets = kAwThreads / kLanes;
    __shared__ float pm[kSets], pl[kSets], pacc[kSets][HD];
    const int tid = threadIdx.x, dl = tid % kLanes, set = tid / kLanes;
    const int head = blockIdx.x, row = blockIdx.y;
    const int b = row / p.n, pos = p.start[b] + (row - b * p.n);
    const size_t q_index = ((size_t)row * p.n_heads + head) * HD;
    const PlaneRef q{const_cast<void *>(p.q), nullptr}, out{p.out, nullptr};
    const float scale = 1.0f / sqrtf((float)HD);
    const int low = p.window > 0 ? max(0, pos - p.window + 1) : 0;
    const int n_first = min(p.sinks, low); // positions in front of the window
    const int count = pos < 0 ? 0 : n_first + pos - low + 1;
    const size_t plane = (size_t)(b * p.n_kv + head / (p.n_heads / p.n_kv)) * p.max_seq_len;

    float qv[8], acc[8] = {}, m = -INFINITY, l = 0.0f;
    plane_load8<QT>(q, q_index + dl * 8, qv);
    for (int j = set; j < count; j += kSets) {
        const int t = j < n_first ? j : low + (j - n_first);
        const size_t at = (plane + cache_row(t, p.max_seq_len, p.sinks)) * HD + dl * 8;
        float kv[8], vv[8], dot = 0.0f;
        plane_load8<CT>(p.cache_k, at, kv);
        plane_load8<CT>(p.cache_v, at, vv);
#pragma unroll
        for (int i = 0; i < 8; i++) dot = fmaf(qv[i], kv[i], dot);
        const float s = group_sum<kLanes>(dot) * scale;
        const float m_new = fmaxf(m, s);
        const float old = m_new > -INFINITY ? expf(m - m_new) : 1.0f, w = m_new > -INFINITY ? expf(s - m_new) : 0.0f;
        m = m_new;
        l = fmaf(l, old, w);
#pragma unroll
        for (int i = 0; i < 8; i++) acc[i] = fmaf(acc[i], old, w * vv[i]);
    }
    if (dl == 0) {
        pm[set] = m;
        pl[set] = l;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) pacc[set][dl * 8 + i] = acc[i];
    __syncthreads();
    if (set != 0) return;
    float top = -INFINITY, total = 0.0f, o[8] = {};
    for (int s = 0; s < kSets; s++) top = fmaxf(top, pm[s]);
    for (int s = 0; s < kSets; s++) {
        if (!(pm[s] > -INFINITY)) continue;
        const float f = expf(pm[s] - top);
        total = fmaf(pl[s], f, total);
#pragma unroll
        for (int i = 0; i < 8; i++) o[i] = fmaf(pacc[s][dl * 8 + i], f, o[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) o[i] = count > 0 ? o[i] / total : 0.0f;
    plane_store8<QT>(out, q_index + dl * 8, o);
}

template <typename QT, typename CT>
static hipError_t launch_window_t(const AttnWindowParams &p, hipStream_t s) {
    const dim3 grid((unsigned)p.n_heads, (unsigned)(p.n * p.n_seqs)), block(kAwThreads);
    switch (p.head_dim) {
    case 32: hipLaunchKernelGGL((attn_window_kernel<QT, CT, 32>), grid, block, 0, s, p); break;
    case 64: hipLaunchKernelGGL((attn_window_kernel<QT, CT, 64>), grid, block, 0, s, p); break;
    case 128: hipLaunchKernelGGL((attn_window_kernel<QT, CT, 128>), grid, block, 0, s, p); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_attn_window(const AttnWindowParams &p, hipStream_t s) {
    if ((int64_t)p.n * p.n_seqs > 65535) return hipErrorInvalidValue;
    switch (p.cache * 2 + p.f16) {
    case kPlaneF16 * 2: return launch_window_t<float, half_t>(p, s);
    case kPlaneF16 * 2 + 1: return launch_window_t<half_t, half_t>(p, s);
    case kPlaneF32 * 2: return launch_window_t<float, float>(p, s);
    case kPlaneF32 * 2 + 1: return launch_window_t<half_t, float>(p, s);
    case kPlaneQ4 * 2: return launch_window_t<float, Quant4>(p, s);
    case kPlaneQ4 * 2 + 1: return launch_window_t<half_t, Quant4>(p, s);
    default: return hipErrorInvalidValue;
    }
}

} // namespace rlh
