// attn_shared.hip -- attention of a batch of texts that share a long prefix.
#include "kernels.h"
#include "answers.h"

namespace rlh {

// One wavefront per row and head, position by position in f32.
template <typename QT, typename CT, int HD>
__global__ __launch_bounds__(64) void attn_shared_kernel(AttnSharedParams p) {
    const int lane = threadIdx.x, row = blockIdx.x, head = blockIdx.y;
    const int b = row / p.n, at = p.start[b] + row - b * p.n, g = head / (p.n_heads / p.n_kv);
    constexpr int kPer = HD > 64 ? HD / 64 : 1;
    QT *out = reinterpret_cast<QT *>(p.out) + ((size_t)row * p.n_heads + head) * HD;
    const QT *q = reinterpret_cast<const QT *>(p.q) + ((size_t)row * p.n_heads + head) * HD;
    float x[kPer], o[kPer], m = -INFINITY, l = 0.0f;
    for (int i = 0; i < kPer; i++) {
        x[i] = lane + 64 * i < HD ? (float)q[lane + 64 * i] : 0.0f;
        o[i] = 0.0f;
    }
    const float scale = 1.0f / sqrtf((float)HD);
    auto see = [&](const PlaneRef &k, const PlaneRef &v, size_t from) {
        float dot = 0.0f;
        for (int i = 0; i < kPer; i++)
            if (lane + 64 * i < HD) dot = fmaf(x[i], plane_load1<CT>(k, from + lane + 64 * i), dot);
        dot = wave_sum(dot) * scale;
        const float m_new = fmaxf(m, dot);
        const float alpha = m > -INFINITY ? expf(m - m_new) : 0.0f, w = m_new > -INFINITY ? expf(dot - m_new) : dot == dot ? 0.0f : dot;
        m = m_new;
        l = l * alpha + w;
        for (int i = 0; i < kPer; i++)
            if (lane + 64 * i < HD) o[i] = o[i] * alpha + (w == 0.0f ? 0.0f : w * plane_load1<CT>(v, from + lane + 64 * i));
    };
    if (at >= 0) {
        for (int t = 0; t < p.prefix_len; t++) see(p.prefix_k, p.prefix_v, ((size_t)g * p.prefix_rows + t) * HD);
        for (int t = 0; t <= at; t++) see(p.cache_k, p.cache_v, (((size_t)b * p.n_kv + g) * p.max_seq_len + t) * HD);
    }
    for (int i = 0; i < kPer; i++)
        if (lane + 64 * i < HD) out[lane + 64 * i] = (QT)(l == 0.0f ? 0.0f : o[i] / l);
}

template <typename QT, typename CT>
static void launch_hd(const AttnSharedParams &p, hipStream_t s) {
    const dim3 grid((unsigned)(p.n * p.n_seqs), (unsigned)p.n_heads);
    if (p.head_dim == 32) hipLaunchKernelGGL((attn_shared_kernel<QT, CT, 32>), grid, dim3(64), 0, s, p);
    else if (p.head_dim == 64) hipLaunchKernelGGL((attn_shared_kernel<QT, CT, 64>), grid, dim3(64), 0, s, p);
    else hipLaunchKernelGGL((attn_shared_kernel<QT, CT, 128>), grid, dim3(64), 0, s, p);
}

hipError_t launch_attn_shared(const AttnSharedParams &p, int compute_units, float *ws, hipStream_t s) {
    switch (p.cache * 2 + p.f16) {
    case kPlaneF16 * 2: launch_hd<float, half_t>(p, s); break;
    case kPlaneF16 * 2 + 1: launch_hd<half_t, half_t>(p, s); break;
    case kPlaneF32 * 2: launch_hd<float, float>(p, s); break;
    case kPlaneF32 * 2 + 1: launch_hd<half_t, float>(p, s); break;
    case kPlaneQ4 * 2: launch_hd<float, Quant4>(p, s); break;
    case kPlaneQ4 * 2 + 1: launch_hd<half_t, Quant4>(p, s); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

} // namespace rlh
