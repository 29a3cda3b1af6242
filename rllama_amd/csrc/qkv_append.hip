// qkv_append.hip -- norms of queries and keys per head, position rotation and cache write in one pass over a projection's rows,
// and the conversion between tensors of 16, 32 and 4 bits.
//
// For a head's vector x of hd values at position t: y = x / sqrt(mean(x^2) + eps) * w, then every pair (a, b) of y becomes
// (a cos - b sin, a sin + b cos) with the angles of position t.  Values go to the cache as they are.
//
// Bound by memory: every element is read once and written once, about 20 operations each.  hd / 8 lanes hold one head's vector,
// 8 consecutive elements per lane: 16-byte accesses, the sum of squares is one exchange over at most 16 lanes, and a 4-bit group is four
// neighbouring lanes, so quantising needs no memory of its own.
//
// Measured: 1500 rows of 32 heads on 8 of 128 into 4 bits, 33 MB: 11.8 to 12.7 us, 2.7 TB/s (a copy of as many bytes: 7.9).  All workgroups are on the part at once, so
// their loads, their arithmetic and their stores come one after the other.  One row of 32 heads: 2.7 us, a launch.
// Call after call, the rows in the caches: 9.0 us; into f16 8.4, 32 key and value heads into f16 13.3.
#include "kernels.h"
#include "longctx.h"

#include <algorithm>

namespace rlh {

constexpr int kAppendThreads = 256;

// eight floats at a 16-byte aligned address
__device__ __forceinline__ void load8(const float *p, float (&v)[8]) {
    const float4_t a = *reinterpret_cast<const float4_t *>(p), b = *reinterpret_cast<const float4_t *>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[i] = a[i];
        v[i + 4] = b[i];
    }
}

// the value of lane i ^ kLanes / 2 of a head's kLanes lanes
template <int kLanes>
__device__ __forceinline__ float other_half(float v) {
    const int x = __builtin_bit_cast(int, v);
    if constexpr (kLanes == 16) return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, x, 0x128 /* row_ror:8 */, 0xf, 0xf, false));
    else if constexpr (kLanes == 8) return __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(x, 0x101f /* xor 4 */));
    else return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, x, kDppQuadPerm2301, 0xf, 0xf, false));
}

// kTake: heads per thread, all of them loaded before the first is worked on.
template <typename IN, typename CT, int HD, int kTake>
__global__ __launch_bounds__(kAppendThreads) void qkv_append_kernel(QkvAppendParams p) {
    constexpr int kLanes = HD / 8, kUnits = kAppendThreads / kLanes;
    const int row = blockIdx.x, b = row / p.n, pos = p.start[b] + (row - b * p.n);
    const int dl = threadIdx.x % kLanes, slots = p.n_heads + 2 * p.n_kv;
    const int first = blockIdx.y * (kUnits * kTake) + threadIdx.x / kLanes;
    const size_t q_row = (size_t)row * p.n_heads * HD + dl * 8;
    if (pos < 0) { // padding: zero queries, nothing in the cache
        const float zero[8] = {};
#pragma unroll
        for (int u = 0; u < kTake; u++)
            if (first + u * kUnits < p.n_heads) plane_store8<IN>(p.q, q_row + (size_t)(first + u * kUnits) * HD, zero);
        return;
    }
    float v[kTake][8];
#pragma unroll
    for (int u = 0; u < kTake; u++) {
        const int slot = min(first + u * kUnits, slots - 1); // (past the last head: read along, not stored)
        plane_load8<IN>(p.qkv, ((size_t)row * slots + slot) * HD + dl * 8, v[u]);
    }
    // the row's angles and the norms' weights, once for all heads that this thread takes
    const float *turn = p.freqs + (size_t)pos * HD;
    float angle[16], qw[8], kw[8]; // neighbouring pairs: (cos, sin) four times; halves: eight cosines, and sines with the sign that this lane's part takes
    const bool second = dl >= kLanes / 2;
    if (p.halves) {
        float lo[8], hi[8];
        load8(turn + dl % (kLanes / 2) * 16, lo);
        load8(turn + dl % (kLanes / 2) * 16 + 8, hi);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            angle[i] = lo[2 * i];
            angle[i + 4] = hi[2 * i];
            angle[i + 8] = second ? lo[2 * i + 1] : -lo[2 * i + 1];
            angle[i + 12] = second ? hi[2 * i + 1] : -hi[2 * i + 1];
        }
    } else {
        float lo[8];
        load8(turn + dl * 8, lo);
#pragma unroll
        for (int i = 0; i < 8; i++) angle[i] = lo[i], angle[i + 8] = 0.0f;
    }
    if (p.q_norm) load8(p.q_norm + dl * 8, qw);
    if (p.k_norm) load8(p.k_norm + dl * 8, kw);
    const size_t cache_at = (size_t)cache_row(pos, p.max_seq_len, p.sinks) * HD + dl * 8;
#pragma unroll
    for (int u = 0; u < kTake; u++) {
        const int slot = first + u * kUnits; // (the lanes of a head stay together)
        if (slot >= slots) break;
        const int kind = slot < p.n_heads ? 0 : slot < p.n_heads + p.n_kv ? 1 : 2; // query, key, value
        if (kind < 2) {
            if (kind == 0 ? p.q_norm != nullptr : p.k_norm != nullptr) {
                float sq = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++) sq = fmaf(v[u][i], v[u][i], sq);
                const float r = rsqrtf(group_sum<kLanes>(sq) / (float)HD + p.eps);
#pragma unroll
                for (int i = 0; i < 8; i++) v[u][i] = v[u][i] * r * (kind == 0 ? qw[i] : kw[i]);
            }
            if (p.halves) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
#pragma clang fp contract(off) // as rope_pair: products and their sum rounded one by one
                    const float other = other_half<kLanes>(v[u][i]);
                    const float own = v[u][i] * angle[i], turned = other * angle[i + 8];
                    v[u][i] = own + turned;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i += 2) rope_pair(v[u][i], v[u][i + 1], make_float2(angle[i], angle[i + 1]), v[u][i], v[u][i + 1]);
            }
        }
        if (kind == 0) {
            plane_store8<IN>(p.q, q_row + (size_t)slot * HD, v[u]);
        } else {
            const int g = slot - p.n_heads - (kind == 2 ? p.n_kv : 0);
            plane_store8<CT>(kind == 1 ? p.cache_k : p.cache_v, (size_t)(b * p.n_kv + g) * p.max_seq_len * HD + cache_at, v[u]);
        }
    }
}

template <typename IN, typename CT, int HD>
static void launch_append(const QkvAppendParams &p, hipStream_t s) {
    const int units = kAppendThreads * 8 / HD, slots = p.n_heads + 2 * p.n_kv, rows = p.n * p.n_seqs;
    // Few workgroups: a head per thread group, so that nothing waits.  More than four per compute unit: three heads, so that angles and weights are read once for them.
    // (1 / 2 / 3 / 4 heads, us a call, 4.2 of it the call; 32 heads on 8 of 128 into f16: 384 rows, 1152 workgroups of one head each, 4.6 / 4.3 / 4.7 / 4.6; 512, 5.2 /
    // 4.7 / 4.7 / 4.7; 1500, 10.9 / 9.8 / 8.4 / 8.4.  32 heads on 32: 256 rows, 1536 workgroups, 5.1 / 4.9 / 5.2 / 5.1; 384, 6.8 / 5.7 / 5.5 / 6.0; 1500, 18.1 / 14.5 / 13.3 /
    // 14.3.  16 of 64 on 16: 768, 1536 workgroups, 4.8 / 4.4 / 4.9 / 4.8; 1500, 7.9 / 6.0 / 6.1 / 6.3.  One workgroup holds all heads of a row, 8 of 32 on 2: 2500 rows 5.1 / 5.4
    // / 5.6 / 5.8.)
    const int groups = (slots + units - 1) / units;
    const int take = groups > 1 && (int64_t)rows * groups > 1024 ? 3 : 1;
    const dim3 grid((unsigned)rows, (unsigned)((slots + units * take - 1) / (units * take)));
    if (take == 1) hipLaunchKernelGGL((qkv_append_kernel<IN, CT, HD, 1>), grid, dim3(kAppendThreads), 0, s, p);
    else hipLaunchKernelGGL((qkv_append_kernel<IN, CT, HD, 3>), grid, dim3(kAppendThreads), 0, s, p);
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
