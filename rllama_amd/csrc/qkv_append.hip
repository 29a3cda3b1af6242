// qkv_append.hip -- norms of queries and keys per head, position rotation and cache write in one pass over a projection's rows,
// and the conversion between tensors of 16, 32 and 4 bits.
//
// For a head's vector x of hd values at position t: y = x / sqrt(mean(x^2) + eps) * w, then every pair (a, b) of y becomes
// (a cos - b sin, a sin + b cos) with the angles of position t.  Values go to the cache as they are.
//
// Bound by memory: every element is read once and written once, about 20 operations each.  hd / 8 lanes hold one head's vector,
// 8 consecutive elements per lane: 16-byte accesses, the sum of squares is one exchange over at most 16 lanes, and a 4-bit group is four
// neighbouring lanes, so quantising needs no memory of its own.
#include "kernels.h"
#include "longctx.h"

#include <algorithm>

namespace rlh {

constexpr int kAppendThreads = 256;

template <typename IN, typename CT, int HD>
__global__ __launch_bounds__(kAppendThreads) void qkv_append_kernel(QkvAppendParams p) {
    constexpr int kLanes = HD / 8, kUnits = kAppendThreads / kLanes;
    const int row = blockIdx.x, b = row / p.n, pos = p.start[b] + (row - b * p.n);
    const int dl = threadIdx.x % kLanes, slots = p.n_heads + 2 * p.n_kv;
    const int first = blockIdx.y * kUnits + threadIdx.x / kLanes, stride = gridDim.y * kUnits;
    const size_t q_row = (size_t)row * p.n_heads * HD + dl * 8;
    if (pos < 0) { // padding: zero queries, nothing in the cache
        const float zero[8] = {};
        for (int slot = first; slot < p.n_heads; slot += stride) plane_store8<IN>(p.q, q_row + (size_t)slot * HD, zero);
        return;
    }
    // the row's angles and the norms' weights, once for all heads that this thread takes
    const float2 *turn = reinterpret_cast<const float2 *>(p.freqs) + (size_t)pos * (HD / 2) + (p.halves ? dl % (kLanes / 2) * 8 : dl * 4);
    const bool second = dl >= kLanes / 2;
    float2 angle[8];
#pragma unroll
    for (int i = 0; i < 8; i++) angle[i] = i < 4 || p.halves ? turn[i] : make_float2(0.0f, 0.0f);
    float qw[8], kw[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        qw[i] = p.q_norm ? p.q_norm[dl * 8 + i] : 1.0f;
        kw[i] = p.k_norm ? p.k_norm[dl * 8 + i] : 1.0f;
    }
    const size_t cache_at = (size_t)cache_row(pos, p.max_seq_len, p.sinks) * HD + dl * 8;
    for (int slot = first; slot < slots; slot += stride) { // (the lanes of a head stay together)
        float v[8];
        plane_load8<IN>(p.qkv, ((size_t)row * slots + slot) * HD + dl * 8, v);
        const int kind = slot < p.n_heads ? 0 : slot < p.n_heads + p.n_kv ? 1 : 2; // query, key, value
        if (kind < 2) {
            if (kind == 0 ? p.q_norm != nullptr : p.k_norm != nullptr) {
                float sq = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) sq = fmaf(v[i], v[i], sq);
                const float r = 1.0f / sqrtf(group_sum<kLanes>(sq) / (float)HD + p.eps);
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = v[i] * r * (kind == 0 ? qw[i] : kw[i]);
            }
            if (p.halves) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float other = __shfl_xor(v[i], kLanes / 2, kLanes);
                    float re, im;
                    rope_pair(second ? other : v[i], second ? v[i] : other, angle[i], re, im);
                    v[i] = second ? im : re;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i += 2) rope_pair(v[i], v[i + 1], angle[i / 2], v[i], v[i + 1]);
            }
        }
        if (kind == 0) {
            plane_store8<IN>(p.q, q_row + (size_t)slot * HD, v);
        } else {
            const int g = slot - p.n_heads - (kind == 2 ? p.n_kv : 0);
            plane_store8<CT>(kind == 1 ? p.cache_k : p.cache_v, (size_t)(b * p.n_kv + g) * p.max_seq_len * HD + cache_at, v);
        }
    }
}

template <typename IN, typename CT, int HD>
static void launch_append(const QkvAppendParams &p, hipStream_t s) {
    const int units = kAppendThreads * 8 / HD, slots = p.n_heads + 2 * p.n_kv, rows = p.n * p.n_seqs;
    // Few rows: a workgroup for every `units` heads of a row, so that nothing waits.  Many rows: one per row, so that angles and weights are read once.
    const int blocks = rows < 512 ? (slots + units - 1) / units : 1;
    hipLaunchKernelGGL((qkv_append_kernel<IN, CT, HD>), dim3((unsigned)rows, (unsigned)blocks), dim3(kAppendThreads), 0, s, p);
}

template <typename IN, typename CT>
static hipError_t launch_append_t(const QkvAppendParams &p, hipStream_t s) {
    switch (p.head_dim) {
    case 32: launch_append<IN, CT, 32>(p, s); break;
    case 64: launch_append<IN, CT, 64>(p, s); break;
    case 128: launch_append<IN, CT, 128>(p, s); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_qkv_append(const QkvAppendParams &p, hipStream_t s) {
    switch (p.cache * 2 + p.f16) {
    case kPlaneF16 * 2: return launch_append_t<float, half_t>(p, s);
    case kPlaneF16 * 2 + 1: return launch_append_t<half_t, half_t>(p, s);
    case kPlaneF32 * 2: return launch_append_t<float, float>(p, s);
    case kPlaneF32 * 2 + 1: return launch_append_t<half_t, float>(p, s);
    case kPlaneQ4 * 2: return launch_append_t<float, Quant4>(p, s);
    case kPlaneQ4 * 2 + 1: return launch_append_t<half_t, Quant4>(p, s);
    default: return hipErrorInvalidValue;
    }
}

// ---- conversion ------------------------------------------------------------------------------------------------------------
template <typename DT, typename ST>
__global__ __launch_bounds__(256) void plane_convert_kernel(PlaneRef dst, PlaneRef src, size_t pieces) {
    // (pieces is a multiple of 4 where the destination has 4 bits: the four lanes of a group stay together)
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (size_t)gridDim.x * 256) {
        float v[8];
        plane_load8<ST>(src, i * 8, v);
        plane_store8<DT>(dst, i * 8, v);
    }
}

hipError_t launch_plane_convert(const PlaneRef &dst, int dst_type, const PlaneRef &src, int src_type, size_t count, hipStream_t s) {
    if (dst_type != kPlaneQ4 && src_type != kPlaneQ4) return launch_convert(dst.data, dst_type == kPlaneF16, src.data, src_type == kPlaneF16, count, s);
    if (count % kQ4Group != 0) return hipErrorInvalidValue;
    const size_t pieces = count / 8;
    const dim3 grid((unsigned)std::min<size_t>((pieces + 255) / 256, 8192)), block(256);
    if (dst_type == kPlaneQ4 && src_type == kPlaneF16) hipLaunchKernelGGL((plane_convert_kernel<Quant4, half_t>), grid, block, 0, s, dst, src, pieces);
    else if (dst_type == kPlaneQ4 && src_type == kPlaneF32) hipLaunchKernelGGL((plane_convert_kernel<Quant4, float>), grid, block, 0, s, dst, src, pieces);
    else if (dst_type == kPlaneF16) hipLaunchKernelGGL((plane_convert_kernel<half_t, Quant4>), grid, block, 0, s, dst, src, pieces);
    else if (dst_type == kPlaneF32) hipLaunchKernelGGL((plane_convert_kernel<float, Quant4>), grid, block, 0, s, dst, src, pieces);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

} // namespace rlh
