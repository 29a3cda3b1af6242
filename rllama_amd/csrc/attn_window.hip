// attn_window.hip -- attention over cache planes of 16, 32 or 4 bits with a sliding window and first tokens that stay visible.
//
// The row at position p sees the positions t <= p with t < sinks or t > p - window:
//   out = sum_t w_t v_t / sum_t w_t,  w_t = exp(q . k_t / sqrt(hd) - m),  m the largest score,
// in one pass over the positions with a running (m, sum w, sum w v) per row.
//
// The rows that share a key and value head (n rows of n_heads / n_kv heads) are taken 16 at a time, so that every cached value is read
// once for all of them and both products go through the matrix cores, transposed so that a row is a column of both:
//   S^T [position x row] = K [position x dim] . q^T,     O^T [dim x row] += V^T [dim x position] . W [position x row]
// With 16 x 16 tiles lane l holds column l % 16 of a result, rows 4 (l / 16) + i: a row's maximum, sum and rescaling factor live in the
// lanes of its column, and the weights a lane has just formed are the operand it has to supply to the second product, if that product's
// inner index runs over the positions in the order 4 h + j (j < 4), 16 + 4 h + j - 4 (h = l / 16).  V then has to be read by position and
// supplied by dimension: a lane loads the hd / 16 neighbouring dims of each of its eight positions (whole rows of V by 16 lanes) and
// transposes them in registers with byte permutes, so cached rows go from memory into registers and nowhere else: no LDS, no barrier in
// the loop.  Tile e of O^T is made of the dims hd / 16 * m + e (m = 0 .. 15).
//
// Two arithmetics.  16 bits: f16 operands, v_mfma_f32_16x16x32_f16, and nothing but the result is rounded to f16.  A weight is the sum of two f16 numbers, 22 bits, and takes
// two products with V (one row behind 383 positions 7.3 -> 7.5 us, 16 texts with a window 16.2 -> 16.5, 65700 positions in 4 bits 27.4 -> 28.1; rounded to f16 the weights left
// 1.6e-4 of the result's size).  A value of 4 bits is 16 * code * (upper part of the scale / 16) + code * (rest) + lowest, two products that f16 holds exactly for every
// scale and a term that is the same for 32 dims, and each goes through the matrix cores by itself.  32 bits: everything in f32 through v_mfma_f32_16x16x4_f32; also
// taken where f16 queries meet an f32 cache, whose values f16 may not hold.
//
// A text is cut into pieces when there are few rows: every workgroup leaves its (m, sum, O) in work memory and a second launch joins them.
//
// Measured: 16 texts, one row each over a window of 1024 and 4, 32 heads on 8 of 128: 63 MB in 13.4 us, 4.7 TB/s, and 3.9 us of join.  5 rows in f32 behind 2107
// positions of 32 heads: 69 MB in 15.0 us, 4.6 TB/s.  Both are bound by memory.  One row behind 65700 positions in 4 bits, 64 heads on 8: 84 MB in 25.8 us,
// 3.3 TB/s: nothing is saturated (vector ALU 43 %, matrix cores 15 %); its 166 registers leave one workgroup to a compute unit, two wavefronts per SIMD, each of which waits for
// the loads of a step 41 % of its time.  One row behind 383 positions, 6.3 MB: 7.6 us, a chain of latencies.
#include "kernels.h"
#include "attn_window_device.h"

#include <algorithm>

namespace rlh {

constexpr int kAwWaves = 8;
constexpr int kAwThreads = kAwWaves * kWave;
constexpr int kAwRows = 16; // rows per workgroup

__device__ __forceinline__ float col_max(float v) { // over the four lanes of a column
    v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float col_sum(float v) {
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) { return __builtin_amdgcn_perm(hi, lo, sel); }
constexpr uint32_t kLoHalves = 0x05040100u, kHiHalves = 0x07060302u; // of (first, second): perm(second, first, .)

template <int kWords>
__device__ __forceinline__ void load_words(uint32_t (&dst)[kWords], buffer_t src, int offset) {
    if constexpr (kWords % 4 == 0) {
#pragma unroll
        for (int w = 0; w < kWords; w += 4) {
            const auto x = __builtin_amdgcn_raw_buffer_load_b128(src, offset + 4 * w, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; i++) dst[w + i] = x[i];
        }
    } else if constexpr (kWords == 2) {
        const auto x = __builtin_amdgcn_raw_buffer_load_b64(src, offset, 0, 0);
        dst[0] = x[0];
        dst[1] = x[1];
    } else {
        static_assert(kWords == 1, "1, 2 or a multiple of 4");
        dst[0] = __builtin_amdgcn_raw_buffer_load_b32(src, offset, 0, 0);
    }
}
// the codes of kN elements (2, 4 or 8)
template <int kN>
__device__ __forceinline__ uint32_t load_codes(buffer_t src, int offset) {
    if constexpr (kN == 8) return __builtin_amdgcn_raw_buffer_load_b32(src, offset, 0, 0);
    else if constexpr (kN == 4) return (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(src, offset, 0, 0);
    else return (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(src, offset, 0, 0);
}
template <typename CT>
constexpr int kElementBits = std::is_same_v<CT, Quant4> ? 4 : (int)sizeof(CT) * 8;

// The operands of one step, and the two products on them.  AC: half_t or float, the arithmetic.
template <typename AC, typename CT, int HD>
struct Step;

// ---- f16 arithmetic, 32 positions --------------------------------------------------------------------------------------------
template <typename CT, int HD>
struct Step<half_t, CT, HD> {
    static constexpr int kPositions = 32;
    static constexpr bool kLowSums = std::is_same_v<CT, Quant4>;
    static constexpr int kTiles = 2;            // of 16 positions
    static constexpr float kLift = kWeightLift;
    static constexpr int kKs = HD / 32;         // MFMAs per score tile
    static constexpr int kDims = HD / 16;       // neighbouring dims of V per lane = tiles of O^T
    static constexpr bool kQ4 = std::is_same_v<CT, Quant4>;
    static constexpr int kBits = kElementBits<CT>;
    struct Queries {
        half8_t q[kKs];
        half8_t sums; // 4 bits: the sum of the lane's dims of q in two f16 parts (the term of the lowest values)
        float up = 1.0f; // what the row's scores are to be multiplied by
    };
    struct Sums { // 4 bits: the lowest values' part of O^T, row m for all dims kDims * m + e; O^T itself is then kept divided by 16
        float4_t low;
    };
    uint32_t k[kTiles][kQ4 ? HD / 32 : HD / 8 /* words: a quarter of a row */];
    uint32_t kp[kTiles];
    uint32_t v[8][kQ4 ? 1 : kDims / 2];
    uint32_t vp[8];

    // lane (row = l % 16, h): dims h * HD / 4 + 8 c .. + 7, in the order of the codes of a word where K has 4 bits
    template <typename QT>
    __device__ static void load_q(Queries &to, const QT *row, int h) {
#pragma unroll
        for (int c = 0; c < kKs; c++) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int d = kQ4 ? (i >> 1) + 4 * (i & 1) : i;
                to.q[c][i] = (half_t)(float)row[h * (HD / 4) + 8 * c + d];
            }
        }
        if constexpr (kQ4) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < HD / 4; i++) sum += (float)row[h * (HD / 4) + i];
            if (col_max(fabsf(sum)) > 65504.0f) { // f16 holds each of the dims but not their sum: the whole row by 2^-6, which is made up for later
                to.up = 64.0f;
                sum *= 0.015625f;
#pragma unroll
                for (int c = 0; c < kKs; c++) to.q[c] *= (half_t)0.015625f;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) to.sums[i] = (half_t)0.0f;
            to.sums[0] = (half_t)sum;
            to.sums[1] = (half_t)(sum - (float)to.sums[0]);
        }
    }
    __device__ void load(buffer_t ck, buffer_t ckp, buffer_t cv, buffer_t cvp, int lane) {
        const int m = lane & 15, h = lane >> 4;
#pragma unroll
        for (int t = 0; t < kTiles; t++) {
            load_words(k[t], ck, (m * HD + h * (HD / 4)) * kBits / 8 + 16 * t * HD * kBits / 8);
            if constexpr (kQ4) kp[t] = __builtin_amdgcn_raw_buffer_load_b32(ckp, (m * HD + h * (HD / 4)) / 32 * 4 + 16 * t * HD / 8, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int row = j < 4 ? j : 12 + j; // + 4 h
            if constexpr (kQ4) {
                v[j][0] = load_codes<kDims>(cv, (4 * h * HD + m * kDims) / 2 + row * HD / 2);
                vp[j] = __builtin_amdgcn_raw_buffer_load_b32(cvp, (4 * h * HD + m * kDims) / 32 * 4 + row * HD / 8, 0, 0);
            } else {
                load_words(v[j], cv, (4 * h * HD + m * kDims) * 2 + row * HD * 2);
            }
        }
    }
    __device__ void scores(const Queries &of, const Q4Bits &bits, float4_t (&s)[kTiles]) const {
        const float4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (kQ4) {
            // codes times either part of the scale, exactly, and the lowest value times the sum of q over the lane's dims: four chains of products
            static_assert(kTiles == 2, "two tiles");
            const Q4Scale scale0(perm(kp[0], kp[0], kLoHalves)), scale1(perm(kp[1], kp[1], kLoHalves));
            auto low_term = [&](uint32_t pair) {
                half8_t a = {};
                a[0] = a[1] = __builtin_bit_cast(half2_t, pair)[1];
                return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, of.sums, zero, 0, 0, 0);
            };
            float4_t s0 = zero, s1 = zero, rest0 = low_term(kp[0]), rest1 = low_term(kp[1]);
            auto add = [&](float4_t &s, float4_t &rest, const Q4Scale &scale, uint32_t word, const half8_t &q) {
                half2_t x[4];
                q4_codes_f16(bits, word, x);
                uint4_t hi, lo;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    hi[i] = __builtin_bit_cast(uint32_t, x[i] * scale.hi16);
                    lo[i] = __builtin_bit_cast(uint32_t, x[i] * scale.lo);
                }
                s = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, hi), q, s, 0, 0, 0);
                rest = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, lo), q, rest, 0, 0, 0);
            };
#pragma unroll
            for (int c = 0; c < kKs; c++) {
                add(s0, rest0, scale0, k[0][c], of.q[c]);
                add(s1, rest1, scale1, k[1][c], of.q[c]);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[0][i] = fmaf(16.0f, s0[i], rest0[i]);
                s[1][i] = fmaf(16.0f, s1[i], rest1[i]);
            }
        } else {
#pragma unroll
            for (int t = 0; t < kTiles; t++) s[t] = zero;
#pragma unroll
            for (int c = 0; c < kKs; c++)
#pragma unroll
                for (int t = 0; t < kTiles; t++)
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, uint4_t{k[t][4 * c], k[t][4 * c + 1], k[t][4 * c + 2], k[t][4 * c + 3]}), of.q[c],
                                                                  s[t], 0, 0, 0);
        }
    }
    // w[t][i]: weights of positions 16 t + 4 h + i
    __device__ void values(const float4_t (&w)[kTiles], const Q4Bits &bits, float4_t (&o)[kDims], Sums &sums) const {
        half8_t b, rest; // a weight is the sum of two f16 numbers
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float x = w[i / 4][i % 4];
            b[i] = (half_t)x;
            rest[i] = (half_t)(x - (float)b[i]);
        }
        if constexpr (kQ4) {
            // positions two by two: the codes of dims 0 .. 3 of both in one word, those of dims 4 .. 7 in another, and each nibble of the pair
            // becomes a pair (first position, second position) of one dim
            half8_t b16; // for the rest of the scales: a part of at most 2^-7 of the value, for which the first number of a weight is enough
#pragma unroll
            for (int i = 0; i < 8; i++) b16[i] = b[i] * (half_t)0.0625f;
            uint4_t low;
#pragma unroll
            for (int j = 0; j < 4; j++) low[j] = perm(vp[2 * j + 1], vp[2 * j], kHiHalves);
            sums.low = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, low), b, sums.low, 0, 0, 0);
            sums.low = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, low), rest, sums.low, 0, 0, 0);
            constexpr int kPart = kDims < 4 ? kDims : 4;
#pragma unroll
            for (int part = 0; part < kDims / kPart; part++) {
                uint4_t hi[kPart], lo[kPart];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const Q4Scale scale(perm(vp[2 * j + 1], vp[2 * j], kLoHalves));
                    half2_t y[4];
                    q4_codes_f16(bits, perm(v[2 * j + 1][0], v[2 * j][0], part ? kHiHalves : kLoHalves), y);
#pragma unroll
                    for (int i = 0; i < kPart; i++) {
                        hi[i][j] = __builtin_bit_cast(uint32_t, y[i] * scale.hi16);
                        lo[i][j] = __builtin_bit_cast(uint32_t, y[i] * scale.lo);
                    }
                }
#pragma unroll
                for (int i = 0; i < kPart; i++) {
                    float4_t &to = o[part * kPart + i];
                    to = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, hi[i]), b, to, 0, 0, 0);
                    to = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, hi[i]), rest, to, 0, 0, 0);
                    to = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, lo[i]), b16, to, 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < kDims; e++) {
                uint4_t a;
#pragma unroll
                for (int j = 0; j < 4; j++) a[j] = perm(v[2 * j + 1][e / 2], v[2 * j][e / 2], e % 2 ? kHiHalves : kLoHalves);
                o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), b, o[e], 0, 0, 0);
                o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), rest, o[e], 0, 0, 0);
            }
        }
    }
    // whether some value of V is not finite
    __device__ bool odd_values() const {
        bool odd = false;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if constexpr (kQ4) {
                odd |= !q4_finite(vp[j]);
            } else {
#pragma unroll
                for (int w = 0; w < kDims / 2; w++) odd |= ((v[j][w] & 0x7c000000u) == 0x7c000000u) || ((v[j][w] & 0x7c00u) == 0x7c00u);
            }
        }
        return odd;
    }
};

// ---- f32 arithmetic, 16 positions --------------------------------------------------------------------------------------------
template <typename CT, int HD>
struct Step<float, CT, HD> {
    static constexpr int kPositions = 16;
    static constexpr bool kLowSums = false;
    static constexpr int kTiles = 1;
    static constexpr float kLift = 0.0f; // (weights stay in f32)
    static constexpr int kDims = HD / 16;
    static constexpr bool kQ4 = std::is_same_v<CT, Quant4>;
    static constexpr int kPerWord = kQ4 ? 8 : std::is_same_v<CT, half_t> ? 2 : 1;
    static constexpr int kKWords = HD / 4 / kPerWord, kVWords = kQ4 ? 1 : kDims / kPerWord;
    struct Queries {
        float q[HD / 4];
        static constexpr float up = 1.0f;
    };
    struct Sums {
        float4_t low; // (of the f16 form)
    };
    // as the cache holds them, so that a load need not have arrived before the next one is issued
    uint32_t k[kKWords], kp, v[4][kVWords], vp[4];

    template <typename QT>
    __device__ static void load_q(Queries &to, const QT *row, int h) {
#pragma unroll
        for (int i = 0; i < HD / 4; i++) to.q[i] = (float)row[h * (HD / 4) + i];
    }
    __device__ void load(buffer_t ck, buffer_t ckp, buffer_t cv, buffer_t cvp, int lane) {
        constexpr int kBits = kElementBits<CT>;
        const int m = lane & 15, h = lane >> 4;
        load_words(k, ck, (m * HD + h * (HD / 4)) * kBits / 8);
        if constexpr (kQ4) kp = __builtin_amdgcn_raw_buffer_load_b32(ckp, (m * HD + h * (HD / 4)) / 32 * 4, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (kQ4) {
                v[i][0] = load_codes<kDims>(cv, (4 * h * HD + m * kDims) / 2 + i * HD / 2);
                vp[i] = __builtin_amdgcn_raw_buffer_load_b32(cvp, (4 * h * HD + m * kDims) / 32 * 4 + i * HD / 8, 0, 0);
            } else {
                load_words(v[i], cv, (4 * h * HD + m * kDims) * (kBits / 8) + i * HD * (kBits / 8));
            }
        }
    }
    template <int kWords>
    __device__ static float value(const uint32_t (&w)[kWords], uint32_t pair, int i) {
        if constexpr (kQ4) return fmaf((float)((w[i / 8] >> (4 * (i % 8))) & 15u), q4_scale(pair), q4_lowest(pair));
        else if constexpr (kPerWord == 2) return (float)__builtin_bit_cast(half2_t, w[i / 2])[i % 2];
        else return __builtin_bit_cast(float, w[i]);
    }
    __device__ void scores(const Queries &of, const Q4Bits &bits, float4_t (&s)[kTiles]) const {
        s[0] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < HD / 4; i++) s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(value(k, kp, i), of.q[i], s[0], 0, 0, 0);
    }
    __device__ void values(const float4_t (&w)[kTiles], const Q4Bits &bits, float4_t (&o)[kDims], Sums &sums) const {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < kDims; e++) o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(value(v[i], vp[i], e), w[0][i], o[e], 0, 0, 0);
    }
    __device__ bool odd_values() const {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < kDims; e++) odd |= !(fabsf(value(v[i], vp[i], e)) <= 3.402823466e38f);
        return odd;
    }
};

template <typename AC, typename QT, typename CT, int HD>
__global__ __launch_bounds__(kAwThreads) void attn_rows_kernel(AttnCutParams pp) {
    typedef Step<AC, CT, HD> St;
    constexpr int kDims = St::kDims, kTiles = St::kTiles, kStep = St::kPositions;
    constexpr int kPad = HD + 4;
    __shared__ float sm[kAwWaves][kAwRows], sl[kAwWaves][kAwRows];
    __shared__ __attribute__((aligned(16))) float so[kAwWaves][kAwRows][kPad];
    const AttnWindowParams &p = pp.a;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int m = lane & 15, h = lane >> 4;
    const int unit = blockIdx.z, tile = blockIdx.y, piece = blockIdx.x;
    const int b = unit / p.n_kv, g = unit - b * p.n_kv;
    const int group = p.n_heads / p.n_kv, rows = p.n * group;
    const int start = p.start[b];
    const int r0 = tile * kAwRows, r1 = min(rows, r0 + kAwRows) - 1;
    const int p0 = max(0, start + r0 / group), p1 = start + r1 / group;

    // the rows' places in q and out: row r is row r / group of the sequence, head g * group + r % group
    const int my_r = min(r0 + m, r1);
    const int my_i = my_r / group;
    const int my_p = r0 + m <= r1 ? start + my_i : -1;

    const int my_low = p.window > 0 ? my_p - p.window + 1 : 0;
    // (bitwise on purpose: with short circuits the compiler made branches of this and lost the masking of a step's first position)
    auto sees = [&](int at, int t_last) { return (bool)((int)(at <= min(my_p, t_last)) & ((int)(at >= my_low) | (int)(at < p.sinks))); };

    Span span = span_of<kStep>(p0, p1, p.window, p.sinks, p.max_seq_len);
    if (p1 < 0) span.steps = 0;
    const int n_pieces = (span.steps + pp.piece_steps - 1) / pp.piece_steps;
    if (piece >= max(1, n_pieces)) return;

    float m_run = -INFINITY, l_run = 0.0f;
    float4_t o[kDims];
#pragma unroll
    for (int e = 0; e < kDims; e++) o[e] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    typename St::Sums sums{float4_t{0.0f, 0.0f, 0.0f, 0.0f}};

    const size_t plane = (size_t)unit * p.max_seq_len;
    typename St::Queries queries;
    St::load_q(queries, reinterpret_cast<const QT *>(p.q) + ((size_t)(b * p.n + my_i) * p.n_heads + g * group + (my_r - my_i * group)) * HD, h);
    const float c2_all = 1.44269504088896340736f / sqrtf((float)HD), c2 = c2_all * queries.up; // (the second one is the row's own)

    struct Place {
        int t0, last, row; // positions t0 .. min(last, t0 + kStep - 1), row of the first one
        bool front;
    };
    auto place_of = [&](int s) {
        if (s < span.steps0) return Place{s * kStep, span.first_end - 1, s * kStep, true};
        if (s < span.steps1) return Place{span.low + (s - span.steps0) * kStep, span.turn - 1, span.row + (s - span.steps0) * kStep, false};
        return Place{span.turn + (s - span.steps1) * kStep, span.last, p.sinks + (s - span.steps1) * kStep, false};
    };
    const Q4Bits bits;
    auto load = [&](St &st, int s) {
        constexpr int kBits = kElementBits<CT>, kRow = HD * kBits / 8, kPairRow = HD / 8;
        const Place at = place_of(s);
        const int rows_here = min(kStep, at.last - at.t0 + 1);
        const size_t row = plane + at.row;
        if constexpr (kBits == 4) {
            st.load(buffer_of(p.cache_k.data, row * kRow, rows_here * kRow), buffer_of(p.cache_k.pairs, row * kPairRow, rows_here * kPairRow),
                    buffer_of(p.cache_v.data, row * kRow, rows_here * kRow), buffer_of(p.cache_v.pairs, row * kPairRow, rows_here * kPairRow), lane);
        } else {
            const buffer_t k = buffer_of(p.cache_k.data, row * kRow, rows_here * kRow), v = buffer_of(p.cache_v.data, row * kRow, rows_here * kRow);
            st.load(k, k, v, v, lane);
        }
    };
    // every row that is no padding sees the whole step?
    auto whole_step = [&](const Place &at) {
        return at.t0 + kStep - 1 <= min(at.last, p0) && (at.front || p.window == 0 || at.t0 > p1 - p.window);
    };
    bool skipped = false, anew = false;
    auto consume = [&](const St &st, int s, auto slow) {
        const Place here = place_of(s);
        const int t0 = here.t0;
        const bool whole = whole_step(here);
        if constexpr (!decltype(slow)::value) { // (see below)
            if (!whole && __any(st.odd_values())) {
                skipped = true;
                return;
            }
        } else if (!anew && !__any(st.odd_values())) {
            return;
        }
        float4_t w[kTiles];
        st.scores(queries, bits, w);
        if (!whole) {
#pragma unroll
            for (int t = 0; t < kTiles; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) w[t][i] = sees(t0 + 16 * t + 4 * h + i, here.last) ? w[t][i] : -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < kTiles; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) top = fmaxf(top, w[t][i]);
        // The reference point of the exponentials follows the maximum only when some row's has grown by more than 2^8 (any point gives the same
        // softmax): weights stay below 2^8 times what they are carried by, and rescaling leaves the common path.
        const float m_new = fmaxf(m_run, col_max(top));
        if (__any((m_new - m_run) * c2 > 8.0f)) { // the first maximum: infinity
            const float alpha = m_run > -INFINITY ? __builtin_amdgcn_exp2f((m_run - m_new) * c2) : 0.0f;
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int e = 0; e < kDims; e++) o[e] *= alpha;
            if constexpr (St::kLowSums) sums.low *= alpha;
        }
        const float mc = (m_run > -INFINITY ? m_run * c2 : 0.0f) - St::kLift;
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < kTiles; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                w[t][i] = __builtin_amdgcn_exp2f(fmaf(w[t][i], c2, -mc));
                sum += w[t][i];
            }
        l_run += sum;
        if constexpr (!decltype(slow)::value) {
            st.values(w, bits, o, sums);
        } else {
#pragma unroll
            for (int t = 0; t < kTiles; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
#pragma unroll 1
                    for (int hh = 0; hh < 4; hh++) {
                        const int j = 16 * t + 4 * hh + i;
                        const float wt = __shfl(w[t][i], hh * 16 + m, kWave) * (St::kLowSums ? 0.0625f : 1.0f);
                        const bool seen = sees(t0 + j, here.last);
                        const size_t from = (plane + here.row + j) * HD + 4 * h * kDims;
#pragma unroll
                        for (int x = 0; x < 4; x++)
#pragma unroll
                            for (int e = 0; e < kDims; e++)
                                if (seen) o[e][x] = fmaf(wt, plane_load1<CT>(p.cache_v, from + x * kDims + e), o[e][x]);
                    }
                }
        }
    };
    // (A second set of operands, loaded ahead, gained nothing at any length and cost 2 to 8 % in f32 for its registers.)
    const int s_end = min(span.steps, (piece + 1) * pp.piece_steps), s_first = piece * pp.piece_steps + wave;
    for (int s = s_first; s < s_end; s += kAwWaves) {
        St st;
        load(st, s);
        consume(st, s, std::false_type{});
    }
    if constexpr (St::kLift != 0.0f) {
        // An infinity that a row sees: the second number of its weight may be 0 or negative, and the sum of both products NaN.
        float odd = 0.0f; // NaN if a sum is not finite
#pragma unroll
        for (int e = 0; e < kDims; e++)
#pragma unroll
            for (int x = 0; x < 4; x++) odd = fmaf(o[e][x], 0.0f, odd);
        anew = __any((int)(odd != 0.0f) & (int)(l_run < INFINITY));
        if (anew) {
            m_run = -INFINITY;
            l_run = 0.0f;
#pragma unroll
            for (int e = 0; e < kDims; e++) o[e] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
            sums.low = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    if (skipped || anew) {
        // Steps that hold a value that is not finite and that some row may not see: in the product its weight 0 would make a NaN of it.
        // Such steps were left out above; here every row adds up what it sees, position by position.  So it does with all steps if some sum is not finite.
        for (int s = s_first; s < s_end; s += kAwWaves) {
            if (!anew && whole_step(place_of(s))) continue;
            St st;
            load(st, s);
            consume(st, s, std::true_type{});
        }
    }

    // ---- join the wavefronts
    l_run = col_sum(l_run);
    if (h == 0) {
        sm[wave][m] = m_run * queries.up;
        sl[wave][m] = l_run;
    }
#pragma unroll
    for (int x = 0; x < 4; x++)
#pragma unroll
        for (int e = 0; e < kDims; e++) so[wave][m][(4 * h + x) * kDims + e] = St::kLowSums ? fmaf(16.0f, o[e][x], sums.low[x]) : o[e][x];
    __syncthreads();
    // thread: row tid / 32, dims HD / 32 of it
    constexpr int kPer = HD / 32;
    const int jr = tid / 32, jd = (tid % 32) * kPer;
    const bool mine = r0 + jr <= r1;
    float M = -INFINITY, L = 0.0f, O[kPer] = {};
#pragma unroll
    for (int w = 0; w < kAwWaves; w++) M = fmaxf(M, sm[w][jr]);
#pragma unroll
    for (int w = 0; w < kAwWaves; w++) {
        if (!(sm[w][jr] > -INFINITY)) { // nothing seen, or only NaN
            L += sl[w][jr];
            continue;
        }
        const float f = __builtin_amdgcn_exp2f((sm[w][jr] - M) * c2_all);
        L = fmaf(sl[w][jr], f, L);
#pragma unroll
        for (int i = 0; i < kPer; i++) O[i] = fmaf(so[w][jr][jd + i], f, O[i]);
    }
    const int jri = (r0 + jr) / group;
    if (start + jri < 0) L = 0.0f; // padding
    QT *out = reinterpret_cast<QT *>(p.out) + ((size_t)(b * p.n + jri) * p.n_heads + g * group + (r0 + jr - jri * group)) * HD + jd;
    if (n_pieces <= 1) {
        if (mine) {
#pragma unroll
            for (int i = 0; i < kPer; i++) out[i] = (QT)(L == 0.0f ? 0.0f : O[i] / L);
        }
        return;
    }
    // ---- leave the piece's (m, sum) and O for attn_join_kernel: of every row first the pairs of all pieces, then the sums
    if (mine) {
        float *ws = pp.ws + ((size_t)unit * rows + r0 + jr) * pp.pieces * (HD + 2);
        if (jd == 0) {
            ws[2 * piece] = M;
            ws[2 * piece + 1] = L;
        }
#pragma unroll
        for (int i = 0; i < kPer; i++) ws[2 * pp.pieces + piece * HD + jd + i] = O[i];
    }
}

template <typename AC, typename QT, typename CT, int HD>
static hipError_t launch_rows(const AttnCutParams &p, hipStream_t s) {
    const int rows = p.a.n * (p.a.n_heads / p.a.n_kv);
    const dim3 grid((unsigned)p.pieces, (unsigned)((rows + kAwRows - 1) / kAwRows), (unsigned)(p.a.n_seqs * p.a.n_kv));
    hipLaunchKernelGGL((attn_rows_kernel<AC, QT, CT, HD>), grid, dim3(kAwThreads), 0, s, p);
    if (p.pieces > 1) launch_attn_join<QT, HD, kAwRows, Step<AC, CT, HD>::kPositions>(p, s);
    return hipGetLastError();
}
template <typename AC, typename QT, typename CT>
static hipError_t launch_rows_hd(const AttnCutParams &p, hipStream_t s) {
    switch (p.a.head_dim) {
    case 32: return launch_rows<AC, QT, CT, 32>(p, s);
    case 64: return launch_rows<AC, QT, CT, 64>(p, s);
    case 128: return launch_rows<AC, QT, CT, 128>(p, s);
    default: return hipErrorInvalidValue;
    }
}

// f32 arithmetic is needed for f32 queries and where an f32 cache may hold what f16 cannot
static bool f16_arithmetic(const AttnWindowParams &p) { return p.f16 && p.cache != kPlaneF32; }

// How the texts are cut: pieces of `piece_steps` steps, at most `pieces` of them; and about what the call takes.
struct RowsCut {
    int pieces, piece_steps;
    int most; // pieces of a text of any length
    double us;
};
static RowsCut cut_rows(const AttnWindowParams &p, int compute_units) {
    const int group = p.n_heads / p.n_kv, step = f16_arithmetic(p) ? 32 : 16;
    const int64_t rows = (int64_t)p.n * group, tiles = (rows + kAwRows - 1) / kAwRows, units = tiles * p.n_seqs * p.n_kv;
    // no tile has more steps than this: its rows' positions are at most `apart` from each other
    const int64_t apart = std::min<int64_t>(p.n - 1, (kAwRows - 2) / group + 1);
    int64_t steps = 1;
    double keys = 0.0; // that an average tile looks at, summed over the sequences
    for (int b = 0; b < p.n_seqs; b++) {
        const int64_t last = (int64_t)p.start[b] + p.n - 1;
        if (last < 0) continue;
        int64_t count = (last + step) / step;
        double mean = 0.5 * (double)(std::max(0, p.start[b]) + last + 1);
        if (p.window > 0) {
            count = std::min(count, (p.window - 1 + apart + step) / step) + (p.sinks + step - 1) / step;
            mean = std::min(mean, (double)p.window + apart + p.sinks);
        }
        if (last >= p.max_seq_len) count++; // the ring's end cuts a step in two
        steps = std::max(steps, count);
        keys += mean;
    }
    // About one workgroup per compute unit, with a step for each wavefront at least.  Up to two and a half steps per wavefront are not cut, nor up to four where there
    // would be two pieces: joining costs a launch, about 3 us (f16, us, whole / cut; 32 heads, one text: 384 positions 7.4 / 8.7 in two pieces, 600: 9.3 / 9.5, 768:
    // 10.5 / 9.7, 1024: 12.0 / 9.7; 16 texts of 8 key and value heads, in two pieces: 600: 9.6 / 11.3, 1000: 13.5 / 13.7).
    const int64_t want = std::max<int64_t>(1, compute_units / units);
    const int64_t n = 2 * steps <= (want == 2 ? 8 : 5) * kAwWaves ? 1 : std::min<int64_t>({want, (steps + kAwWaves - 1) / kAwWaves, kMaxPieces});
    RowsCut cut;
    cut.most = (int)std::min<int64_t>(want, kMaxPieces);
    cut.piece_steps = (int)((steps + n - 1) / n);
    cut.pieces = (int)((steps + cut.piece_steps - 1) / cut.piece_steps);
    cut.us = 5.0 + (cut.pieces > 1 ? 3.5 : 0.0) + units * 0.01 + tiles * p.n_kv * keys * p.head_dim / 128 * 30e-6 + (double)cut.piece_steps * step * p.head_dim / 128 * 4e-3;
    return cut;
}

// The tiles of attn_tiles.hip take 128 rows at once, this kernel 16: it reads K and V once per 16 rows, but has more workgroups, no second rounding of 4-bit values
// and more wavefronts per key.  Both sides' estimates were fitted to measured shapes (17 .. 2400 rows per key and value head, 0 .. 8000 positions, f16 and 4 bits);
// over 262 of them going by the estimates costs 1.5 % over always taking the faster one, 60 % at worst, a fixed limit of 64 rows 11 to 13 %, 140 at worst.  (us, this / tiles, 32 heads of 128: 128 rows from position 0
// 7.1 / 8.8, behind 500 14.9 / 20.0, behind 2000 41 / 21.7; 64 rows behind 4000 44 / 22.)
static bool tiles_take(const AttnWindowParams &p, int compute_units) {
    return f16_arithmetic(p) && !p.exact && p.n * (int64_t)(p.n_heads / p.n_kv) > kAwRows && attn_tiles_us(p, compute_units) < cut_rows(p, compute_units).us;
}

int64_t attn_window_most_rows(const AttnWindowParams &p, int compute_units) {
    if ((int64_t)p.n_seqs * p.n_kv > 65535) return 0;
    return 65535 * (int64_t)(tiles_take(p, compute_units) ? attn_tiles_rows() : kAwRows);
}

size_t attn_window_work_floats(const AttnWindowParams &p, int compute_units) {
    if (tiles_take(p, compute_units)) return attn_tiles_work_floats(p, compute_units);
    const RowsCut cut = cut_rows(p, compute_units);
    return cut.pieces > 1 ? (size_t)p.n * p.n_heads * p.n_seqs * cut.most * (p.head_dim + 2) : 0;
}

hipError_t launch_attn_window(const AttnWindowParams &a, int compute_units, float *ws, hipStream_t s) {
    if (tiles_take(a, compute_units)) return launch_attn_tiles(a, compute_units, ws, s);
    AttnCutParams p;
    p.a = a;
    p.ws = ws;
    const RowsCut cut = cut_rows(a, compute_units);
    p.pieces = cut.pieces;
    p.piece_steps = cut.piece_steps;
    switch (a.cache * 2 + a.f16) {
    case kPlaneF16 * 2: return launch_rows_hd<float, float, half_t>(p, s);
    case kPlaneF16 * 2 + 1: return launch_rows_hd<half_t, half_t, half_t>(p, s);
    case kPlaneF32 * 2: return launch_rows_hd<float, float, float>(p, s);
    case kPlaneF32 * 2 + 1: return launch_rows_hd<float, half_t, float>(p, s);
    case kPlaneQ4 * 2: return launch_rows_hd<float, float, Quant4>(p, s);
    case kPlaneQ4 * 2 + 1: return launch_rows_hd<half_t, half_t, Quant4>(p, s);
    default: return hipErrorInvalidValue;
    }
}

} // namespace rlh
