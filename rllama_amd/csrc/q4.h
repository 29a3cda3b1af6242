// q4.h -- tensors of 4 bits (RLH_Q4) and cache planes of any type as the kernels see them.
//
// A 4-bit tensor of `count` elements is one buffer: count / 2 bytes of codes (element 2 i in the low half of byte i), then one 32-bit word
// for every group of 32 elements: the f16 scale in the low half, the f16 lowest value in the high half.  Codes and pairs are planes of
// their own so that both are read in whole aligned words: 32 codes are 16 bytes, and a row's pairs lie side by side.
#pragma once

#include "device_utils.h"

namespace rlh {

struct Quant4 {}; // tag of the storage type
constexpr int kQ4Group = 32;

inline size_t q4_pairs_offset(size_t count) { return count / 2; }

// One plane: where the elements are and, for 4 bits, where the pairs are.
struct PlaneRef {
    void *data;
    uint32_t *pairs;
};

// The row of the cache that holds position t (max_seq_len rows; positions past them replace the oldest behind the first `sinks`)
__host__ __device__ inline int cache_row(int t, int max_seq_len, int sinks) { return t < max_seq_len ? t : sinks + (t - sinks) % (max_seq_len - sinks); }

__device__ __forceinline__ float q4_scale(uint32_t pair) { return (float)__builtin_bit_cast(half2_t, pair)[0]; }
__device__ __forceinline__ float q4_lowest(uint32_t pair) { return (float)__builtin_bit_cast(half2_t, pair)[1]; }

template <int kCtrl>
__device__ __forceinline__ float quad_perm(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kCtrl, 0xf, 0xf, false));
}

// Pair and codes of a group of 32 values held by four neighbouring lanes, eight consecutive ones each: the lane's codes; every lane
// of the four gets the pair.
__device__ __forceinline__ uint32_t q4_encode8(const float (&v)[8], uint32_t &pair) {
    float mn = v[0], mx = v[0], odd = 0.0f; // odd: NaN if some value is not finite
#pragma unroll
    for (int i = 0; i < 8; i++) {
        mn = fminf(mn, v[i]);
        mx = fmaxf(mx, v[i]);
        odd += v[i] - v[i];
    }
    mn = fminf(mn, quad_perm<kDppQuadPerm1032>(mn));
    mn = fminf(mn, quad_perm<kDppQuadPerm2301>(mn));
    mx = fmaxf(mx, quad_perm<kDppQuadPerm1032>(mx));
    mx = fmaxf(mx, quad_perm<kDppQuadPerm2301>(mx));
    odd = group_sum<4>(odd);
    half_t low = to_f16(mn + 0.0f); // (zeros of either kind are positive: which of two zeros fminf gives is open)
    half_t scale = to_f16((mx - (float)low + 0.0f) / 15.0f);
    const float check = odd + ((float)low - (float)low) + ((float)scale - (float)scale); // 0, or NaN: the group reads as NaN
    uint32_t codes = 0;
    if (!(check == 0.0f)) {
        pair = 0x7e000000u;
        return codes;
    }
    pair = (uint32_t)__builtin_bit_cast(uint16_t, scale) | ((uint32_t)__builtin_bit_cast(uint16_t, low) << 16);
    const float s = (float)scale, l = (float)low;
    if (s > 0.0f) {
        // (v - l) / s rounded to a whole number, by the reciprocal: within 2^-19 of the quotient up to 16 (two roundings), so only next to a tie is the quotient itself needed
        const float inv = 1.0f / s;
        bool tie = false;
        float c[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float t = (v[i] - l) * inv;
            c[i] = rintf(t);
            tie |= fabsf(fabsf(t - c[i]) - 0.5f) < 1e-5f;
        }
        if (tie) {
#pragma unroll
            for (int i = 0; i < 8; i++) c[i] = rintf((v[i] - l) / s);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) codes |= (uint32_t)fminf(fmaxf(c[i], 0.0f), 15.0f) << (4 * i);
    }
    return codes;
}

__device__ __forceinline__ void q4_decode8(uint32_t codes, uint32_t pair, float (&v)[8]) {
    const float s = q4_scale(pair), l = q4_lowest(pair);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = fmaf((float)((codes >> (4 * i)) & 15u), s, l);
}

// Eight consecutive elements, index a multiple of 8, of a plane or a tensor of type T as floats and back.  For 4 bits the four lanes of a group
// store together.
template <typename T>
__device__ __forceinline__ void plane_load8(const PlaneRef &p, size_t index, float (&v)[8]) {
    if constexpr (std::is_same_v<T, Quant4>) {
        q4_decode8(reinterpret_cast<const uint32_t *>(p.data)[index / 8], p.pairs[index / kQ4Group], v);
    } else if constexpr (sizeof(T) == 2) {
        const half8_t h = *reinterpret_cast<const half8_t *>(reinterpret_cast<const half_t *>(p.data) + index);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (float)h[i];
    } else {
        const float4_t a = *reinterpret_cast<const float4_t *>(reinterpret_cast<const float *>(p.data) + index);
        const float4_t b = *reinterpret_cast<const float4_t *>(reinterpret_cast<const float *>(p.data) + index + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[i] = a[i];
            v[i + 4] = b[i];
        }
    }
}
template <typename T>
__device__ __forceinline__ void plane_store8(const PlaneRef &p, size_t index, const float (&v)[8]) {
    if constexpr (std::is_same_v<T, Quant4>) {
        uint32_t pair;
        reinterpret_cast<uint32_t *>(p.data)[index / 8] = q4_encode8(v, pair);
        if (index % kQ4Group == 0) p.pairs[index / kQ4Group] = pair;
    } else if constexpr (sizeof(T) == 2) {
        half8_t h;
#pragma unroll
        for (int i = 0; i < 8; i++) h[i] = to_f16(v[i]);
        *reinterpret_cast<half8_t *>(reinterpret_cast<half_t *>(p.data) + index) = h;
    } else {
        float4_t a, b;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            a[i] = v[i];
            b[i] = v[i + 4];
        }
        *reinterpret_cast<float4_t *>(reinterpret_cast<float *>(p.data) + index) = a;
        *reinterpret_cast<float4_t *>(reinterpret_cast<float *>(p.data) + index + 4) = b;
    }
}

} // namespace rlh
