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
// Two arithmetics.  16 bits: f16 operands, v_mfma_f32_16x16x32_f16; weights are rounded to f16, as are values of 4 bits (each half a
// unit in the eleventh bit, and neither adds up over a text).  32 bits: everything in f32 through v_mfma_f32_16x16x4_f32; also taken where f16
// queries meet an f32 cache, whose values f16 may not hold.
//
// A text is cut into pieces when there are few rows: every workgroup leaves its (m, sum, O) in work memory and the last one to
// arrive joins them, in the order of the pieces.
#include "kernels.h"
#include "longctx.h"

#include <algorithm>

namespace rlh {

constexpr int kAwWaves = 8;
constexpr int kAwThreads = kAwWaves * kWave;
constexpr int kAwRows = 16; // rows per workgroup

// What one workgroup's rows look at: steps of kStep positions, first the tokens that stay visible, then the window.
struct Span {
    int first_end;   // positions 0 .. first_end - 1 are looked at through `sinks`
    int low, last;   // and low .. last
    int first_steps, steps;
};
template <int kStep>
__host__ __device__ inline Span span_of(int p0, int p1, int window, int sinks) { // positions of the first and the last row that is no padding
    Span s;
    s.low = window > 0 ? (p0 - window + 1 > 0 ? p0 - window + 1 : 0) : 0;
    s.last = p1;
    s.first_end = sinks < s.low ? sinks : s.low;
    s.first_steps = (s.first_end + kStep - 1) / kStep;
    s.steps = s.first_steps + (s.last - s.low + kStep) / kStep;
    return s;
}

__device__ __forceinline__ float col_max(float v) { // over the four lanes of a column
    v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float col_sum(float v) {
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}

// eight codes of a word as f16 numbers lowest + code * scale: pairs (0, 4), (1, 5), (2, 6), (3, 7).  1024 + c is the f16 number with c in its
// last bits (0x6400 | c); 1024 + 16 c likewise, which saves half of the shifts.  The difference to 1024 is exact, the multiply-add rounds once.
__device__ __forceinline__ void q4_pairs_f16(uint32_t w, half2_t scale, half2_t scale16, half2_t low, half2_t (&out)[4]) {
    const half2_t k1024 = {(half_t)1024.0f, (half_t)1024.0f};
#pragma unroll
    for (int s = 0; s < 2; s++) {
        const uint32_t x = w >> (8 * s);
        const half2_t a = __builtin_bit_cast(half2_t, (x & 0x000f000fu) | 0x64006400u) - k1024;
        const half2_t b = __builtin_bit_cast(half2_t, (x & 0x00f000f0u) | 0x64006400u) - k1024;
        out[2 * s] = __builtin_elementwise_fma(a, scale, low);
        out[2 * s + 1] = __builtin_elementwise_fma(b, scale16, low);
    }
}
__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) { return __builtin_amdgcn_perm(hi, lo, sel); }
constexpr uint32_t kLoHalves = 0x05040100u, kHiHalves = 0x07060302u; // of (first, second): perm(second, first, .)

// The operands of one step, and the two products on them.  AC: half_t or float, the arithmetic.
template <typename AC, typename CT, int HD>
struct Step;

// ---- f16 arithmetic, 32 positions --------------------------------------------------------------------------------------------
template <typename CT, int HD>
struct Step<half_t, CT, HD> {
    static constexpr int kPositions = 32;
    static constexpr int kTiles = 2;            // of 16 positions
    static constexpr int kKs = HD / 32;         // MFMAs per score tile
    static constexpr int kDims = HD / 16;       // neighbouring dims of V per lane = tiles of O^T
    static constexpr bool kQ4 = std::is_same_v<CT, Quant4>;
    half8_t q[kKs];
    uint32_t k[kTiles][kQ4 ? HD / 32 : HD / 8 /* words: a quarter of a row */];
    uint32_t kp[kTiles];
    uint32_t v[8][kQ4 ? 1 : kDims / 2];
    uint32_t vp[8];

    // lane (row = l % 16, h): dims h * HD / 4 + 8 c .. + 7, in the order of the codes of a word where K has 4 bits
    template <typename QT>
    __device__ void load_q(const QT *row, int h) {
#pragma unroll
        for (int c = 0; c < kKs; c++) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int d = kQ4 ? (i >> 1) + 4 * (i & 1) : i;
                q[c][i] = (half_t)(float)row[h * (HD / 4) + 8 * c + d];
            }
        }
    }
    template <int kWords>
    __device__ static void load_words(uint32_t (&dst)[kWords], const void *src) {
        if constexpr (kWords % 4 == 0) {
#pragma unroll
            for (int w = 0; w < kWords; w += 4) {
                const uint4_t x = *reinterpret_cast<const uint4_t *>(reinterpret_cast<const uint32_t *>(src) + w);
#pragma unroll
                for (int i = 0; i < 4; i++) dst[w + i] = x[i];
            }
        } else if constexpr (kWords == 2) {
            const uint2 x = *reinterpret_cast<const uint2 *>(src);
            dst[0] = x.x;
            dst[1] = x.y;
        } else {
            dst[0] = *reinterpret_cast<const uint32_t *>(src);
        }
    }
    // row_of(j): the plane's row of the step's position j
    template <typename F>
    __device__ void load(const PlaneRef &ck, const PlaneRef &cv, int lane, F row_of) {
        const int m = lane & 15, h = lane >> 4;
#pragma unroll
        for (int t = 0; t < kTiles; t++) {
            const size_t at = (size_t)row_of(16 * t + m) * HD + h * (HD / 4);
            if constexpr (kQ4) {
                load_words(k[t], reinterpret_cast<const char *>(ck.data) + at / 2);
                kp[t] = ck.pairs[at / 32];
            } else {
                load_words(k[t], reinterpret_cast<const char *>(ck.data) + at * 2);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const size_t at = (size_t)row_of(j < 4 ? 4 * h + j : 12 + 4 * h + j) * HD + m * kDims;
            if constexpr (kQ4) {
                v[j][0] = kDims == 8   ? reinterpret_cast<const uint32_t *>(cv.data)[at / 8]
                          : kDims == 4 ? (uint32_t)reinterpret_cast<const uint16_t *>(cv.data)[at / 4]
                                       : (uint32_t)reinterpret_cast<const uint8_t *>(cv.data)[at / 2];
                vp[j] = cv.pairs[at / 32];
            } else {
                load_words(v[j], reinterpret_cast<const char *>(cv.data) + at * 2);
            }
        }
    }
    __device__ void scores(float4_t (&s)[kTiles]) const {
#pragma unroll
        for (int t = 0; t < kTiles; t++) {
            s[t] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
            half2_t scale, scale16, low;
            if constexpr (kQ4) {
                scale = __builtin_bit_cast(half2_t, perm(kp[t], kp[t], kLoHalves));
                low = __builtin_bit_cast(half2_t, perm(kp[t], kp[t], kHiHalves));
                scale16 = scale * half2_t{(half_t)0.0625f, (half_t)0.0625f};
            }
#pragma unroll
            for (int c = 0; c < kKs; c++) {
                half8_t a;
                if constexpr (kQ4) {
                    half2_t x[4];
                    q4_pairs_f16(k[t][c], scale, scale16, low, x);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        a[2 * i] = x[i][0];
                        a[2 * i + 1] = x[i][1];
                    }
                } else {
                    a = __builtin_bit_cast(half8_t, uint4_t{k[t][4 * c], k[t][4 * c + 1], k[t][4 * c + 2], k[t][4 * c + 3]});
                }
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, q[c], s[t], 0, 0, 0);
            }
        }
    }
    // w[t][i]: weights of positions 16 t + 4 h + i
    __device__ void values(const float4_t (&w)[kTiles], float4_t (&o)[kDims]) const {
        half8_t b;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            b[i] = (half_t)w[0][i];
            b[i + 4] = (half_t)w[1][i];
        }
        if constexpr (kQ4) {
            // positions two by two: the codes of dims 0 .. 3 of both in one word, those of dims 4 .. 7 in another, and each nibble of the pair
            // becomes a pair (first position, second position) of one dim
            uint32_t x[kDims][4];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const half2_t scale = __builtin_bit_cast(half2_t, perm(vp[j + 1], vp[j], kLoHalves)), low = __builtin_bit_cast(half2_t, perm(vp[j + 1], vp[j], kHiHalves));
                const half2_t scale16 = scale * half2_t{(half_t)0.0625f, (half_t)0.0625f};
#pragma unroll
                for (int part = 0; part < (kDims + 3) / 4; part++) {
                    half2_t y[4];
                    q4_pairs_f16(perm(v[j + 1][0], v[j][0], part ? kHiHalves : kLoHalves), scale, scale16, low, y);
#pragma unroll
                    for (int i = 0; i < (kDims < 4 ? kDims : 4); i++) x[4 * part + i][j / 2] = __builtin_bit_cast(uint32_t, y[i]);
                }
            }
#pragma unroll
            for (int e = 0; e < kDims; e++)
                o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, uint4_t{x[e][0], x[e][1], x[e][2], x[e][3]}), b, o[e], 0, 0, 0);
        } else {
#pragma unroll
            for (int e = 0; e < kDims; e++) {
                uint4_t a;
#pragma unroll
                for (int j = 0; j < 4; j++) a[j] = perm(v[2 * j + 1][e / 2], v[2 * j][e / 2], e % 2 ? kHiHalves : kLoHalves);
                o[e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), b, o[e], 0, 0, 0);
            }
        }
    }
    // whether some value of V is not finite
    __device__ bool odd_values() const {
        bool odd = false;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if constexpr (kQ4) {
                odd |= ((vp[j] & 0x7c000000u) == 0x7c000000u) || ((vp[j] & 0x7c00u) == 0x7c00u);
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
    static constexpr int kTiles = 1;
    static constexpr int kDims = HD / 16;
    float q[HD / 4], k[HD / 4], v[4][kDims];

    template <typename QT>
    __device__ void load_q(const QT *row, int h) {
#pragma unroll
        for (int i = 0; i < HD / 4; i++) q[i] = (float)row[h * (HD / 4) + i];
    }
    template <int kN>
    __device__ static void load_values(float (&dst)[kN], const PlaneRef &p, size_t at) {
        if constexpr (std::is_same_v<CT, Quant4>) {
            const uint32_t pair = p.pairs[at / 32];
            const float s = q4_scale(pair), l = q4_lowest(pair);
            uint32_t w = 0;
#pragma unroll
            for (int i = 0; i < kN; i++) {
                if (i % 8 == 0)
                    w = kN >= 8   ? reinterpret_cast<const uint32_t *>(p.data)[(at + i) / 8]
                        : kN == 4 ? (uint32_t)reinterpret_cast<const uint16_t *>(p.data)[at / 4]
                                  : (uint32_t)reinterpret_cast<const uint8_t *>(p.data)[at / 2];
                dst[i] = fmaf((float)((w >> (4 * (i % 8))) & 15u), s, l);
            }
        } else {
            const CT *src = reinterpret_cast<const CT *>(p.data) + at;
            constexpr int kPer = 16 / sizeof(CT) < kN ? 16 / sizeof(CT) : kN;
            typedef __attribute__((ext_vector_type(kPer))) CT vec_t;
#pragma unroll
            for (int i = 0; i < kN; i += kPer) {
                const vec_t x = *reinterpret_cast<const vec_t *>(src + i);
#pragma unroll
                for (int j = 0; j < kPer; j++) dst[i + j] = (float)x[j];
            }
        }
    }
    template <typename F>
    __device__ void load(const PlaneRef &ck, const PlaneRef &cv, int lane, F row_of) {
        const int m = lane & 15, h = lane >> 4;
        load_values(k, ck, (size_t)row_of(m) * HD + h * (HD / 4));
#pragma unroll
        for (int i = 0; i < 4; i++) load_values(v[i], cv, (size_t)row_of(4 * h + i) * HD + m * kDims);
    }
    __device__ void scores(float4_t (&s)[kTiles]) const {
        s[0] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < HD / 4; i++) s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[i], q[i], s[0], 0, 0, 0);
    }
    __device__ void values(const float4_t (&w)[kTiles], float4_t (&o)[kDims]) const {
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < kDims; e++) o[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][e], w[0][i], o[e], 0, 0, 0);
    }
    __device__ bool odd_values() const {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < kDims; e++) odd |= !(fabsf(v[i][e]) <= 3.402823466e38f);
        return odd;
    }
};

template <typename T>
__device__ __forceinline__ float plane_load1(const PlaneRef &p, size_t at) {
    if constexpr (std::is_same_v<T, Quant4>) {
        const uint32_t pair = p.pairs[at / 32], c = (reinterpret_cast<const uint8_t *>(p.data)[at / 2] >> (4 * (at & 1))) & 15u;
        return fmaf((float)c, q4_scale(pair), q4_lowest(pair));
    } else {
        return (float)reinterpret_cast<const T *>(p.data)[at];
    }
}

struct AttnRowsParams {
    AttnWindowParams a;
    float *ws;
    unsigned *tickets;
    int pieces, piece_steps;
};

template <typename AC, typename QT, typename CT, int HD>
__global__ __launch_bounds__(kAwThreads) void attn_rows_kernel(AttnRowsParams pp) {
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

    Span span = span_of<kStep>(p0, p1, p.window, p.sinks);
    if (p1 < 0) span.steps = 0;
    const int n_pieces = (span.steps + pp.piece_steps - 1) / pp.piece_steps;
    if (piece >= max(1, n_pieces)) return;

    float m_run = -INFINITY, l_run = 0.0f;
    float4_t o[kDims];
#pragma unroll
    for (int e = 0; e < kDims; e++) o[e] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};

    const size_t plane = (size_t)unit * p.max_seq_len;
    const float c2 = 1.44269504088896340736f / sqrtf((float)HD);
    const int ring = p.max_seq_len - p.sinks;
    St st;
    st.load_q(reinterpret_cast<const QT *>(p.q) + ((size_t)(b * p.n + my_i) * p.n_heads + g * group + (my_r - my_i * group)) * HD, h);

    const int s_end = min(span.steps, (piece + 1) * pp.piece_steps);
    for (int s = piece * pp.piece_steps + wave; s < s_end; s += kAwWaves) {
        const bool front = s < span.first_steps;
        const int t0 = front ? s * kStep : span.low + (s - span.first_steps) * kStep;
        const int t_last = front ? span.first_end - 1 : span.last;
        const int base = cache_row(t0, p.max_seq_len, p.sinks);
        // positions past the end read the last one's row
        auto row_of = [&](int j) {
            int r = base + min(j, t_last - t0);
            if (r >= p.max_seq_len) r -= ring;
            return plane + r;
        };
        st.load(p.cache_k, p.cache_v, lane, row_of);
        float4_t w[kTiles];
        st.scores(w);
        // every row sees the whole step?
        const bool whole = t0 + kStep - 1 <= min(t_last, p0) && start + r0 / group >= 0 && (front || p.window == 0 || t0 > p1 - p.window);
        if (!whole) {
#pragma unroll
            for (int t = 0; t < kTiles; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int at = t0 + 16 * t + 4 * h + i;
                    w[t][i] = sees(at, t_last) ? w[t][i] : -INFINITY;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < kTiles; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) top = fmaxf(top, w[t][i]);
        const float m_new = fmaxf(m_run, col_max(top));
        const float mc = m_new > -INFINITY ? m_new * c2 : 0.0f;
        const float alpha = __builtin_amdgcn_exp2f(fmaf(m_run, c2, -mc)); // nothing seen so far: exp2(-inf) = 0
        m_run = m_new;
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < kTiles; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                w[t][i] = __builtin_amdgcn_exp2f(fmaf(w[t][i], c2, -mc));
                sum += w[t][i];
            }
        l_run = fmaf(l_run, alpha, sum);
#pragma unroll
        for (int e = 0; e < kDims; e++) o[e] *= alpha;
        if (!whole && __any(st.odd_values())) {
            // a value that is not finite and that some row may not see: its weight 0 would still make a NaN of it in the product
#pragma unroll
            for (int t = 0; t < kTiles; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
#pragma unroll 1
                    for (int hh = 0; hh < 4; hh++) {
                        const int j = 16 * t + 4 * hh + i, at = t0 + j;
                        const float wt = __shfl(w[t][i], hh * 16 + m, kWave);
                        const bool seen = sees(at, t_last);
                        const size_t from = (size_t)row_of(j) * HD + 4 * h * kDims;
#pragma unroll
                        for (int x = 0; x < 4; x++)
#pragma unroll
                            for (int e = 0; e < kDims; e++)
                                if (seen) o[e][x] = fmaf(wt, plane_load1<CT>(p.cache_v, from + x * kDims + e), o[e][x]);
                    }
                }
        } else {
            st.values(w, o);
        }
    }

    // ---- join the wavefronts
    l_run = col_sum(l_run);
    if (h == 0) {
        sm[wave][m] = m_run;
        sl[wave][m] = l_run;
    }
#pragma unroll
    for (int x = 0; x < 4; x++)
#pragma unroll
        for (int e = 0; e < kDims; e++) so[wave][m][(4 * h + x) * kDims + e] = o[e][x];
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
        const float f = __builtin_amdgcn_exp2f((sm[w][jr] - M) * c2);
        L = fmaf(sl[w][jr], f, L);
#pragma unroll
        for (int i = 0; i < kPer; i++) O[i] = fmaf(so[w][jr][jd + i], f, O[i]);
    }
    const int jri = (r0 + jr) / group;
    QT *out = reinterpret_cast<QT *>(p.out) + ((size_t)(b * p.n + jri) * p.n_heads + g * group + (r0 + jr - jri * group)) * HD + jd;
    if (n_pieces <= 1) {
        if (mine) {
#pragma unroll
            for (int i = 0; i < kPer; i++) out[i] = (QT)(L == 0.0f ? 0.0f : O[i] / L);
        }
        return;
    }
    // ---- join the pieces
    __shared__ int is_last;
    const size_t slot = (size_t)unit * gridDim.y + tile;
    float *ws = pp.ws + slot * pp.pieces * (kAwRows * (HD + 2));
    auto put = [](float *dst, float v) { __hip_atomic_store(dst, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    auto get = [](const float *src) { return __hip_atomic_load(src, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    float *own = ws + (size_t)piece * (kAwRows * (HD + 2)) + jr * (HD + 2);
    if (mine) {
        if (jd == 0) {
            put(own, M);
            put(own + 1, L);
        }
#pragma unroll
        for (int i = 0; i < kPer; i++) put(own + 2 + jd + i, O[i]);
    }
    // Device-scope stores go through this part's L2s and device-scope loads miss them, so a store that has been acknowledged is seen by
    // the workgroup that draws the last ticket (a property of gfx950; rlh_init refuses every other part).
    asm volatile("" ::: "memory");
    wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    __syncthreads();
    if (tid == 0) {
        const unsigned before = __hip_atomic_fetch_add(pp.tickets + slot, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        is_last = before == (unsigned)(n_pieces - 1);
        if (is_last) __hip_atomic_store(pp.tickets + slot, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); // ready for the next launch
    }
    __syncthreads();
    if (!is_last || !mine) return;
    const float *from = ws + jr * (HD + 2);
    M = -INFINITY;
    L = 0.0f;
    for (int s = 0; s < n_pieces; s++) M = fmaxf(M, get(from + (size_t)s * (kAwRows * (HD + 2))));
#pragma unroll
    for (int i = 0; i < kPer; i++) O[i] = 0.0f;
    for (int s = 0; s < n_pieces; s++) {
        const float *x = from + (size_t)s * (kAwRows * (HD + 2));
        const float ms = get(x), ls = get(x + 1);
        const float f = ms > -INFINITY ? __builtin_amdgcn_exp2f((ms - M) * c2) : 0.0f;
        L += ms > -INFINITY ? ls * f : ls;
#pragma unroll
        for (int i = 0; i < kPer; i++) O[i] = fmaf(f > 0.0f ? get(x + 2 + jd + i) : 0.0f, f, O[i]);
    }
#pragma unroll
    for (int i = 0; i < kPer; i++) out[i] = (QT)(L == 0.0f ? 0.0f : O[i] / L);
}

template <typename AC, typename QT, typename CT, int HD>
static hipError_t launch_rows(const AttnRowsParams &p, hipStream_t s) {
    const int rows = p.a.n * (p.a.n_heads / p.a.n_kv);
    const dim3 grid((unsigned)p.pieces, (unsigned)((rows + kAwRows - 1) / kAwRows), (unsigned)(p.a.n_seqs * p.a.n_kv));
    hipLaunchKernelGGL((attn_rows_kernel<AC, QT, CT, HD>), grid, dim3(kAwThreads), 0, s, p);
    return hipGetLastError();
}
template <typename AC, typename QT, typename CT>
static hipError_t launch_rows_hd(const AttnRowsParams &p, hipStream_t s) {
    switch (p.a.head_dim) {
    case 32: return launch_rows<AC, QT, CT, 32>(p, s);
    case 64: return launch_rows<AC, QT, CT, 64>(p, s);
    case 128: return launch_rows<AC, QT, CT, 128>(p, s);
    default: return hipErrorInvalidValue;
    }
}

// f32 arithmetic is needed for f32 queries and where an f32 cache may hold what f16 cannot
static bool f16_arithmetic(const AttnWindowParams &p) { return p.f16 && p.cache != kPlaneF32; }

// How the texts are cut: pieces of `piece_steps` steps, at most `pieces` of them.
static void cut_rows(const AttnWindowParams &p, int compute_units, int *pieces, int *piece_steps) {
    const int group = p.n_heads / p.n_kv, rows = p.n * group, step = f16_arithmetic(p) ? 32 : 16;
    const int64_t units = (int64_t)((rows + kAwRows - 1) / kAwRows) * p.n_seqs * p.n_kv;
    // no tile has more steps than this: its rows' positions are at most `apart` from each other
    const int64_t apart = std::min<int64_t>(p.n - 1, (kAwRows - 2) / group + 1);
    int64_t steps = 1;
    for (int b = 0; b < p.n_seqs; b++) {
        const int64_t last = (int64_t)p.start[b] + p.n - 1;
        if (last < 0) continue;
        int64_t count = (last + step) / step;
        if (p.window > 0) count = std::min(count, (p.window - 1 + apart + step) / step) + (p.sinks + step - 1) / step;
        steps = std::max(steps, count);
    }
    const int64_t want = std::max<int64_t>(1, 2 * compute_units / units);
    const int64_t n = std::min<int64_t>({want, (steps + kAwWaves - 1) / kAwWaves, 64});
    *piece_steps = (int)((steps + n - 1) / n);
    *pieces = (int)((steps + *piece_steps - 1) / *piece_steps);
}

void attn_window_work(const AttnWindowParams &p, int compute_units, size_t *floats, size_t *tickets) {
    int pieces, piece_steps;
    cut_rows(p, compute_units, &pieces, &piece_steps);
    const int rows = p.n * (p.n_heads / p.n_kv);
    const size_t slots = (size_t)((rows + kAwRows - 1) / kAwRows) * p.n_seqs * p.n_kv;
    *tickets = pieces > 1 ? slots : 0;
    *floats = pieces > 1 ? slots * pieces * kAwRows * (p.head_dim + 2) : 0;
}

hipError_t launch_attn_window(const AttnWindowParams &a, int compute_units, float *ws, unsigned *tickets, hipStream_t s) {
    AttnRowsParams p;
    p.a = a;
    p.ws = ws;
    p.tickets = tickets;
    cut_rows(a, compute_units, &p.pieces, &p.piece_steps);
    if ((int64_t)a.n_seqs * a.n_kv > 65535 || (int64_t)a.n * (a.n_heads / a.n_kv) > 65535 * kAwRows) return hipErrorInvalidValue;
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
