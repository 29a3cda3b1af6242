// attn_window_device.h -- what the two kernels of rlh_attn_window share: the span of positions a workgroup looks at, loads through buffer
// descriptors, and the conversion of 4-bit codes to f16.
#pragma once

#include "longctx.h"

namespace rlh {

// What one workgroup's rows look at, in steps of kStep positions that lie side by side in the cache: the first tokens that stay visible,
// the window up to the end of the ring, the rest of the window from the ring's beginning.
struct Span {
    int first_end;  // positions 0 .. first_end - 1 are looked at through `sinks`
    int low, last;  // and low .. last
    int row, turn;  // row of position low; the first position behind the ring's end (last + 1 if none is)
    int steps0, steps1, steps;
};
template <int kStep>
__device__ inline Span span_of(int p0, int p1, int window, int sinks, int max_seq_len) { // positions of the first and the last row that is no padding
    Span s;
    s.low = window > 0 ? max(0, p0 - window + 1) : 0;
    s.last = p1;
    s.first_end = min(sinks, s.low);
    s.row = cache_row(s.low, max_seq_len, sinks);
    const int room = max_seq_len - s.row; // (all of low .. last fit the ring, so they pass its end once at most)
    s.turn = s.last - s.low < room ? s.last + 1 : s.low + room;
    s.steps0 = (s.first_end + kStep - 1) / kStep;
    s.steps1 = s.steps0 + (s.turn - s.low + kStep - 1) / kStep;
    s.steps = s.steps1 + (s.last + 1 - s.turn + kStep - 1) / kStep;
    return s;
}

// Loads through a buffer descriptor of the step's rows: offsets per lane that never change, one scalar base per step, and rows past the step's
// last one read as zeros by the hardware's bounds check, whatever memory holds there.
typedef __amdgpu_buffer_rsrc_t buffer_t;
__device__ __forceinline__ buffer_t buffer_of(const void *data, size_t offset, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(reinterpret_cast<const char *>(data)) + offset, 0, bytes, 0x00027000);
}
// Masks and exponent bits of the conversion below, kept in registers: masking and setting the exponent are one instruction then, which takes
// no literals and one scalar register at most.
struct Q4Bits {
    uint32_t even = 0x000f000fu, odd = 0x00f000f0u, exp_even = 0x64006400u, exp_odd = 0x54005400u;
    __device__ Q4Bits() {
        asm("" : "+s"(even));
        asm("" : "+s"(odd));
        asm("" : "+v"(exp_even));
        asm("" : "+v"(exp_odd));
    }
};
// eight codes of a word as f16 numbers: pairs (0, 4), (1, 5), (2, 6), (3, 7).  1024 + c is the f16 number with c in its last four bits
// (0x6400 | c), 64 + c the one with c four bits further up (0x5400 | 16 c), which saves half of the shifts.  The differences are exact.
__device__ __forceinline__ void q4_codes_f16(const Q4Bits &bits, uint32_t w, half2_t (&out)[4]) {
    const half2_t k1024 = {(half_t)1024.0f, (half_t)1024.0f}, k64 = {(half_t)64.0f, (half_t)64.0f};
#pragma unroll
    for (int s = 0; s < 2; s++) {
        const uint32_t x = w >> (8 * s);
        out[2 * s] = __builtin_bit_cast(half2_t, (x & bits.even) | bits.exp_even) - k1024;
        out[2 * s + 1] = __builtin_bit_cast(half2_t, (x & bits.odd) | bits.exp_odd) - k64;
    }
}
// the values, lowest + code * scale, each rounded once
__device__ __forceinline__ void q4_pairs_f16(const Q4Bits &bits, uint32_t w, half2_t scale, half2_t low, half2_t (&out)[4]) {
    q4_codes_f16(bits, w, out);
#pragma unroll
    for (int i = 0; i < 4; i++) out[i] = __builtin_elementwise_fma(out[i], scale, low);
}
// A scale as a sum of its upper seven bits and the rest: products of either part with a code have at most eleven bits, so f16 holds them exactly.
// The upper part comes divided by 16: f16 holds that too (its last bit is 16 units of the scale's), and 15 codes of it for every scale there is.
struct Q4Scale {
    half2_t hi16, lo;
    __device__ explicit Q4Scale(uint32_t scales) {
        const half2_t hi = __builtin_bit_cast(half2_t, scales & 0xfff0fff0u);
        hi16 = hi * half2_t{(half_t)0.0625f, (half_t)0.0625f};
        lo = __builtin_bit_cast(half2_t, scales) - hi;
    }
};
// whether scale and lowest value of a group are finite
__device__ __forceinline__ bool q4_finite(uint32_t pair) { return (int)((pair & 0x7c000000u) != 0x7c000000u) & (int)((pair & 0x7c00u) != 0x7c00u); }

// Weights that go through the matrix cores in f16 are carried this power of two larger: the largest is 2^7, and 2^15 while the reference point lags.  Behind a first token that takes
// most of the weight the others are small; below 2^-14 f16 has fewer than eleven bits and the sum in f32 would keep what the products lose (6000 positions with
// 0.2 % of the weight: 7e-3 of the result).  So n weights lose n 2^-32 of the result at most to that.
constexpr float kWeightLift = 7.0f;

// A text that is cut: work memory, for every row first the pairs (m, sum) of its pieces and then the sums O of each, and how it is cut.
struct AttnCutParams {
    AttnWindowParams a;
    float *ws;
    int pieces, piece_steps; // pieces of `piece_steps` steps, at most `pieces` of them
};
constexpr int kMaxPieces = 64;
// Rows of K and V planes from `row` on.
struct PlaneRows {
    PlaneRef k, v;
    size_t row;
};
// How the kernels see a call of rlh_attn_window: its parameters, the position of a sequence's row i, and where a row's partial results go.  rlh_attn_shared has another one.
struct WindowView {
    static constexpr bool kTexts = false; // see attn_rows_device.h
    static constexpr int first_slot = 0;  // of the pieces' places in work memory
    const AttnWindowParams &p;
    float *const &ws; // (references, to what a kernel reads from its arguments where it needs it: with copies, which lived through the loops, f16 heads of 64 took 93 registers instead of
    const int &pieces, &piece_steps; // 80, and two workgroups fitted a compute unit instead of three)
    __device__ explicit WindowView(const AttnCutParams &c) : p(c.a), ws(c.ws), pieces(c.pieces), piece_steps(c.piece_steps) {}
    __device__ int start(int b) const { return p.start[b]; }
    __device__ int position(int start, int i) const { return start + i; }
    __device__ constexpr bool partial() const { return false; } // whether results are left for a join whatever the number of pieces
    __device__ int text(int) const { return 0; }
    __device__ PlaneRows planes(int unit, int, int row) const { return {p.cache_k, p.cache_v, (size_t)unit * p.max_seq_len + row}; }
    __device__ float *partials(int unit, int rows, int r, int hd) const { return ws + ((size_t)unit * rows + r) * pieces * (hd + 2); }
};

// Joins the pieces of rows: weights exp(m_s - M) of all pieces of a row at once (a lane each), then the sums, added up in the same order whatever
// arrives when.  kShare wavefronts take a row: four where there are few rows, one where there are many (a workgroup for each of 32768 rows took 40 us).
// A launch of its own: joining by the last workgroup to arrive took 5.7 us behind pieces of 1000 positions and 11 us behind 32 pieces of 2000
// (device-scope stores, ticket and loads, one after the other), this takes about 3.
constexpr int kAjWaves = 4;

// One row: `ws` holds the pairs (m, sum) of `slots` pieces and then their sums O; the first n_pieces count.  All threads of the workgroup take part.  out(): where the row's
// result goes, worked out behind the sums, which the loads have to be on their way for first.
template <typename QT, int HD, int kShare, typename Out>
__device__ __forceinline__ void join_pieces(float (&part)[kAjWaves * (kWave / (HD / 2))][HD], const float *ws, int slots, int n_pieces, Out out) {
    constexpr int kLanes = HD / 2, kSub = kWave / kLanes; // lanes per piece, pieces side by side in a wavefront
    constexpr int kParts = kShare * kSub;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const float c2 = 1.44269504088896340736f / sqrtf((float)HD);
    // the first sums are on their way before their weights are known
    const int sub = lane / kLanes, d = (lane % kLanes) * 2, s_first = (wave % kShare) * kSub + sub;
    constexpr int kBatch = 4;
    float2 x[kBatch];
    auto fetch = [&](int s0) {
#pragma unroll
        for (int u = 0; u < kBatch; u++) x[u] = *reinterpret_cast<const float2 *>(ws + 2 * slots + (size_t)min(s0 + u * kParts, n_pieces - 1) * HD + d);
    };
    fetch(s_first);
    float m = -INFINITY, l = 0.0f;
    if (lane < n_pieces) {
        m = ws[2 * lane];
        l = ws[2 * lane + 1];
    }
    const float M = wave_max(m);
    const float f = m > -INFINITY ? __builtin_amdgcn_exp2f((m - M) * c2) : 0.0f;
    const float L = wave_sum(m > -INFINITY ? l * f : l); // (nothing seen: 0; only NaN: NaN)
    float2 o = make_float2(0.0f, 0.0f);
    for (int s0 = s_first; s0 - sub < n_pieces; s0 += kParts * kBatch) {
        if (s0 != s_first) fetch(s0);
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
            const int s = s0 + u * kParts;
            const float fs = __shfl(f, min(s, kWave - 1), kWave);
            if (s < n_pieces && fs > 0.0f) {
                o.x = fmaf(x[u].x, fs, o.x);
                o.y = fmaf(x[u].y, fs, o.y);
            }
        }
    }
    *reinterpret_cast<float2 *>(&part[wave * kSub + sub][d]) = o;
    __syncthreads();
    QT *const to = out();
    for (int e = kShare == 1 ? lane : (int)threadIdx.x; e < HD; e += kShare * kWave) {
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kParts; w++) sum += part[wave / kShare * kParts + w][e];
        to[e] = (QT)(L == 0.0f ? 0.0f : sum / L);
    }
}

template <typename QT, int HD, int kTileRows, int kStep, int kShare>
__global__ __launch_bounds__(kAjWaves *kWave) void attn_join_kernel(AttnCutParams pp) {
    __shared__ float part[kAjWaves * (kWave / (HD / 2))][HD];
    const AttnWindowParams &p = pp.a;
    const int wave = threadIdx.x / kWave;
    const int group = p.n_heads / p.n_kv, rows = p.n * group;
    const int unit = blockIdx.y, b = unit / p.n_kv, g = unit - b * p.n_kv, start = p.start[b];
    const int r = blockIdx.x * (kAjWaves / kShare) + wave / kShare; // (with four wavefronts per row all of them leave together below)
    int n_pieces = 0;
    if (r < rows) {
        const int r0 = r / kTileRows * kTileRows, r1 = min(rows, r0 + kTileRows) - 1;
        const Span span = span_of<kStep>(max(0, start + r0 / group), start + r1 / group, p.window, p.sinks, p.max_seq_len);
        n_pieces = start + r1 / group < 0 ? 0 : (span.steps + pp.piece_steps - 1) / pp.piece_steps;
    }
    if (n_pieces <= 1) { // the row is finished
        if constexpr (kShare == 1) __syncthreads();
        return;
    }
    join_pieces<QT, HD, kShare>(part, pp.ws + ((size_t)unit * rows + r) * pp.pieces * (HD + 2), pp.pieces, n_pieces, [&] {
        const int i = r / group;
        return reinterpret_cast<QT *>(p.out) + ((size_t)(b * p.n + i) * p.n_heads + g * group + (r - i * group)) * HD;
    });
}

template <typename QT, int HD, int kTileRows, int kStep>
inline void launch_attn_join(const AttnCutParams &p, hipStream_t s) {
    const unsigned rows = (unsigned)(p.a.n * (p.a.n_heads / p.a.n_kv)), units = (unsigned)(p.a.n_seqs * p.a.n_kv);
    if ((int64_t)rows * units <= 1024) hipLaunchKernelGGL((attn_join_kernel<QT, HD, kTileRows, kStep, kAjWaves>), dim3(rows, units), dim3(kAjWaves * kWave), 0, s, p);
    else hipLaunchKernelGGL((attn_join_kernel<QT, HD, kTileRows, kStep, 1>), dim3((rows + kAjWaves - 1) / kAjWaves, units), dim3(kAjWaves * kWave), 0, s, p);
}

} // namespace rlh
