// attn_tiles_device.h -- rlh_attn_window and rlh_attn_shared for many rows, as a function of one workgroup: f16 arithmetic, tiles of keys staged in LDS.
//
// Workgroup = four row groups of 32 rows on one key and value head (row r = row r / group of the sequence, head r % group of the group), a wavefront for each,
// or two of them that share the keys.  The keys the rows look at pass by in tiles of 64 per wavefront, K and V as f16 in two LDS stages: the next tile is on
// its way while this one is used, one barrier per tile.  f16 caches go from memory straight into LDS; of 4-bit caches a thread takes whole groups of 32
// codes, converts them in registers and writes 64 bytes, so a code is converted once per workgroup and not once per wavefront.
//
// Rounded to f16: the softmax's weights, as operands of the second product, and 4-bit values when they are converted (lowest + code * scale, one rounding of at most
// 2^-11 of the value, where the codes themselves are off by 1/30 of a group's range).  Random values, a window of 1024: the result is off by 4.6e-4 of its size, 2.6e-4
// with an f16 cache, 2.1e-4 with nothing but the result rounded, as in the form for few rows.  Weights as sums of two f16 numbers alone took 57 -> 78 us (2048 rows of 40
// heads) and 51 -> 61 (1500 rows with a window over 4 bits, then 4.1e-4); values of 4 bits would take a second product each besides.
//
// Tiles that every row of the wavefront sees whole, in the middle of a run of rows that lie side by side in the cache, go through a loop of their own with
// nothing but running addresses between the products.  (2048 rows behind 2000 positions, 32 heads of 128 on 8: 133 us with the place of every tile and its
// masks worked out anew, 119 so.)
//
// Measured: 2048 rows from position 0, 40 heads of 128, 43 GFLOP: 56 us, 765 TFLOP/s; 2048 rows behind 2000 positions, 32 heads on 8, 101 GFLOP: 112 us, 900 (a large
// library product reaches 1190).  The matrix cores are busy for 34 % of the first, the vector ALU for 38 %: texts from position 0 give workgroups of 2 to 32 tiles, so that on
// average 1.3 wavefronts of two per SIMD are there, which wait for 23 % of their time.
//
// Both products run transposed through v_mfma_f32_32x32x16_f16, so that a row is a lane pair's column of both results:
//   S^T [key x row] = K . q^T,   O^T [dim x row] += V^T . W
// Register v of lane l holds row 8 (v / 4) + 4 (l / 32) + v % 4 of a result, column l % 32.  The weights a lane has just formed are the second product's
// operand when its inner index runs over the keys in that order: slot i of half h in 16-key slab s is key 16 s + 8 (i / 4) + 4 h + i % 4, i.e.
// two runs of four keys.  ds_read_b64_tr_b16 delivers exactly such a run: of a 4 x 16 block (16 lanes, lane i addressing 4 columns of row i / 4) lane i
// receives column i's four rows.  V therefore stays in LDS as the cache has it, one key per row.
//
// LDS places.  Rows of K: the 16-byte pieces of row r are permuted by r, so that eight consecutive rows' pieces of one column lie in different banks.  Rows of V:
// 64-byte blocks are permuted by r so that the four rows of a transposing read do.
#pragma once

#include "attn_window_device.h"

namespace rlh {

typedef __attribute__((ext_vector_type(16))) float float16_t;
typedef __attribute__((ext_vector_type(4))) _Float16 half4_t;
typedef __attribute__((ext_vector_type(4))) short short4_t;
typedef __attribute__((ext_vector_type(2))) unsigned short ushort2_t;

// The value of lane i ^ 32.  (Written out: of the builtin's two results the compiler kept one where both operands are the same value.)
__device__ __forceinline__ float other_half_lane(float v) {
    float a = v, b = v; // afterwards lanes 32 .. 63 of a hold lanes 0 .. 31 of v, and lanes 0 .. 31 of b hold lanes 32 .. 63
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
    return (threadIdx.x & 32) ? a : b;
}

constexpr int kAtGroups = 4; // of 32 rows
constexpr int kAtRows = 32 * kAtGroups;

// LDS of a workgroup, kShares wavefronts per row group
template <int HD, int kShares>
struct TilesShared {
    static constexpr int kTileBytes = 64 * kShares * HD * 2, kJoinFloats = (HD / 2 + 2) * 64, kOutRow = HD + 8; // K or V of a tile; O, m and sum of a wavefront; padded row of the output tile, halves
    static constexpr int kEndBytes = kShares > 1 ? kAtGroups * kJoinFloats * 4 : kAtGroups * 32 * kOutRow * 2;
    static constexpr int kBytes = 4 * kTileBytes > kEndBytes ? 4 * kTileBytes : kEndBytes;
};

// Row block `block` (128 rows) of unit b * n_kv + g, piece `piece` of their positions.  View: see attn_window_device.h; View::kTexts: the unit is a key and value head, its
// rows are those of all texts, and the tiles are the shared prefix's and then those of every text's own positions, which that text's rows see.
template <typename CT, int HD, int kShares, typename View>
__device__ __forceinline__ void attn_tiles(const View &v, unsigned char *lds, int &sh_wide, int unit, int block, int piece) {
    constexpr bool kQ4 = std::is_same_v<CT, Quant4>;
    constexpr int kWaves = kAtGroups * kShares, kRows = kAtRows;
    constexpr int kAtKeys = 64 * kShares;        // per tile
    constexpr int kKS = HD / 16;                 // MFMA steps over the head dimension
    constexpr int kDT = HD / 32;                 // 32-dim tiles of O^T
    constexpr int kPieces = HD / 8;              // 16-byte pieces per row
    constexpr int kRowBytes = HD * 2;
    typedef TilesShared<HD, kShares> Lds;
    constexpr int kTileBytes = Lds::kTileBytes, kStageBytes = 2 * kTileBytes, kOutRow = Lds::kOutRow, kJoinFloats = Lds::kJoinFloats;
    static_assert(kTileBytes == kAtKeys * kRowBytes, "K or V of a tile");
    static_assert(32 * kOutRow * 2 <= kJoinFloats * 4, "a row group's output goes where its join was");
    const auto &p = v.p; // (sh_wide: 4 bits: some group of the tiles holds a value that is infinity in f16)
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int rg = wave % kAtGroups, kh = wave / kAtGroups; // row group, half of the keys
    const int b = View::kTexts ? 0 : unit / p.n_kv, g = unit - b * p.n_kv;
    const int group = p.n_heads / p.n_kv, rows = p.n * group, start = v.start(b);
    const int r0 = block * kRows, r1 = min(rows, r0 + kRows) - 1;
    const int p0 = max(0, v.position(start, r0 / group)), p1 = v.position(start, r1 / group); // (kTexts: these and the next two are not used)
    // this wavefront's rows, and this lane's
    const int w0 = r0 + rg * 32, w1 = min(r1, w0 + 31);
    const int wp0 = v.position(start, View::kTexts ? 0 : w0 / group), wp1 = w1 < w0 ? -1 : v.position(start, w1 / group);
    const int my_r = min(w0 + col, r1), my_i = my_r / group;
    const int my_p = w0 + col <= r1 ? v.position(start, my_i) : -1;
    const int my_low = p.window > 0 ? max(0, my_p - p.window + 1) : 0;
    const int my_text = w0 + col <= r1 ? v.text(my_i) : -1, first_text = v.text(min(w0, r1) / group), last_text = v.text(w1 / group); // this lane's, this wavefront's
    const half_t *q_row = reinterpret_cast<const half_t *>(p.q) + ((size_t)(b * p.n + my_i) * p.n_heads + g * group + (my_r - my_i * group)) * HD;

    // q as the second operand: lane supplies dims 16 ks + 8 half .. + 7, in the order of the converted codes where the cache has 4 bits
    half8_t q[kKS];
#pragma unroll
    for (int ks = 0; ks < kKS; ks++) {
        const half8_t x = *reinterpret_cast<const half8_t *>(q_row + ks * 16 + half * 8);
#pragma unroll
        for (int i = 0; i < 8; i++) q[ks][i] = x[kQ4 ? (i >> 1) + 4 * (i & 1) : i];
    }
    float16_t o[kDT];
#pragma unroll
    for (int d = 0; d < kDT; d++)
#pragma unroll
        for (int v = 0; v < 16; v++) o[d][v] = 0.0f;
    float m_run = -INFINITY, l_run = 0.0f;

    auto span = [&] {
        if constexpr (View::kTexts) {
            return v.template walk<kAtKeys>(r0, r1, lane);
        } else {
            Span s = span_of<kAtKeys>(p0, p1, p.window, p.sinks, p.max_seq_len);
            if (p1 < 0) s.steps = 0;
            return s;
        }
    }();
    // (texts are cut into pieces with two wavefronts per row group only)
    const int n_pieces = kShares > 1 ? (span.steps + v.piece_steps - 1) / v.piece_steps : 1;
    if (piece >= max(1, n_pieces)) return;
    const int s_first = kShares > 1 ? piece * v.piece_steps : 0, s_end = kShares > 1 ? min(span.steps, s_first + v.piece_steps) : span.steps;
    const float c2 = 1.44269504088896340736f / sqrtf((float)HD);
    const unsigned lds_base = (unsigned)(uintptr_t)(__attribute__((address_space(3))) void *)lds;

    struct Place {
        int t0, last, row;
        bool front;
        int text = -1; // kTexts: whose positions they are; the prefix's: -1
    };
    auto place_of = [&](int s) {
        if constexpr (View::kTexts) {
            const auto at = span.at(s);
            return Place{at.t0, at.last, at.t0, false, at.text};
        } else {
            if (s < span.steps0) return Place{s * kAtKeys, span.first_end - 1, s * kAtKeys, true};
            if (s < span.steps1) return Place{span.low + (s - span.steps0) * kAtKeys, span.turn - 1, span.row + (s - span.steps0) * kAtKeys, false};
            return Place{span.turn + (s - span.steps1) * kAtKeys, span.last, p.sinks + (s - span.steps1) * kAtKeys, false};
        }
    };
    auto planes_of = [&](const Place &at) { return v.planes(unit, at.text, at.row); };
    auto k_swz = [](int row) { return kPieces >= 16 ? row & 15 : (row / (16 / kPieces)) & (kPieces - 1); };
    auto v_swz = [](int row) { return HD == 128 ? (row & 3) * 4 : HD == 64 ? ((row >> 1) & 1) * 4 : 0; }; // in pieces

    // ---- staging
    constexpr int kIssues = kTileBytes / (kWaves * 1024);    // f16: wavefront-wide 1 KiB loads per tile of K (and of V)
    constexpr int kIssueRows = kWaves * 64 / kPieces;        // rows from one to the next: a multiple of what the permutations repeat after
    constexpr int kGroups = 2 * kAtKeys * HD / 32, kItems = kGroups / (64 * kWaves) > 0 ? kGroups / (64 * kWaves) : 1; // 4 bits: groups per tile, and per thread
    static_assert(kTileBytes == kIssues * kWaves * 1024 && 2 * kIssues == kKS, "whole loads of every wavefront, one beside each step of the first product");
    const int my_row = (wave * 64 + lane) / kPieces, my_piece = lane % kPieces;
    const unsigned k_from = (my_piece ^ k_swz(my_row)) << 4, v_from = (my_piece ^ v_swz(my_row)) << 4; // within the row
    uint32_t codes[kQ4 ? kItems : 1][4], pairs[kQ4 ? kItems : 1];
    // `here` rows: f16 on their way to a stage, codes on their way to registers
    auto fetch = [&](const PlaneRows &planes, int here, unsigned stage) __attribute__((always_inline)) {
        const size_t row = planes.row;
        if constexpr (kQ4) {
            const buffer_t k = buffer_of(planes.k.data, row * (HD / 2), here * (HD / 2)), kp = buffer_of(planes.k.pairs, row * (HD / 8), here * (HD / 8));
            const buffer_t v = buffer_of(planes.v.data, row * (HD / 2), here * (HD / 2)), vp = buffer_of(planes.v.pairs, row * (HD / 8), here * (HD / 8));
#pragma unroll
            for (int i = 0; i < kItems; i++) {
                const int item = i * 64 * kWaves + tid, at_group = item % (kGroups / 2); // row at_group / (HD / 32), group at_group % (HD / 32)
                const bool is_v = kItems > 1 ? i >= kItems / 2 : (__builtin_amdgcn_readfirstlane(item / (kGroups / 2)) & 1);
                const auto x = is_v ? __builtin_amdgcn_raw_buffer_load_b128(v, at_group * 16, 0, 0) : __builtin_amdgcn_raw_buffer_load_b128(k, at_group * 16, 0, 0);
#pragma unroll
                for (int w = 0; w < 4; w++) codes[i][w] = x[w];
                pairs[i] = is_v ? __builtin_amdgcn_raw_buffer_load_b32(vp, at_group * 4, 0, 0) : __builtin_amdgcn_raw_buffer_load_b32(kp, at_group * 4, 0, 0);
            }
        } else {
            const half_t *k = reinterpret_cast<const half_t *>(planes.k.data) + row * HD, *v = reinterpret_cast<const half_t *>(planes.v.data) + row * HD;
#pragma unroll
            for (int i = 0; i < kIssues; i++) {
                const unsigned from = (unsigned)min(my_row + i * kIssueRows, here - 1) * kRowBytes; // keys past the last one are masked below
                const unsigned to = lds_base + stage * kStageBytes + (unsigned)(i * kWaves + wave) * 1024u;
                dma16_base(k, from + k_from, to);
                dma16_base(v, from + v_from, to + kTileBytes);
            }
        }
    };
    const Q4Bits bits;
    bool wide = false;
    // 4 bits: word w of the fetched codes (eight of them) as f16 into a stage
    auto place_word = [&](unsigned stage, int word) __attribute__((always_inline)) {
        const int i = word / 4, w = word % 4;
        const unsigned item = i * 64 * kWaves + (unsigned)tid;
        if (kGroups < 64 * kWaves && item >= kGroups) return;
        const unsigned at_group = item % (kGroups / 2), r = at_group / (HD / 32), c = at_group % (HD / 32) * 4 + w;
        const bool is_v = item >= kGroups / 2;
        const half2_t pair = __builtin_bit_cast(half2_t, pairs[i]), scale = {pair[0], pair[0]}, low = {pair[1], pair[1]};
        if (w == 0) wide |= __builtin_fabsf16(__builtin_fmaf16((half_t)15.0f, pair[0], pair[1])) == (half_t)INFINITY;
        half2_t x[4];
        q4_pairs_f16(bits, codes[i][w], scale, low, x);
        uint4_t y;
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = __builtin_bit_cast(uint32_t, x[j]);
        *reinterpret_cast<uint4_t *>(lds + stage * kStageBytes + (is_v ? kTileBytes : 0) + r * kRowBytes + ((c ^ (is_v ? v_swz(r) : k_swz(r))) << 4)) = y;
    };
    auto place = [&](unsigned stage) __attribute__((always_inline)) {
        if constexpr (kQ4) {
#pragma unroll
            for (int word = 0; word < 4 * kItems; word++) place_word(stage, word);
        }
    };

    // the last position of a place that this lane's row may see
    auto limit_of = [&](const Place &at) {
        if constexpr (View::kTexts) return at.text < 0 ? at.last : at.text == my_text ? min(my_p, at.last) : -1;
        else return min(my_p, at.last);
    };
    auto sees = [&](int at, int limit) { return (bool)((int)(at <= limit) & ((int)(at >= my_low) | (int)(at < p.sinks))); };
    auto whole_to = [&](const Place &at) { // up to which every row of the wavefront sees a place
        if constexpr (View::kTexts) return at.text < 0 ? at.last : -1;
        else return min(at.last, max(0, wp0));
    };
    // of this wavefront's half of a tile: every row that is no padding sees all of it / none sees any of it
    auto whole_half = [&](const Place &at) {
        const int t0 = at.t0 + kh * 64;
        return t0 + 63 <= whole_to(at) && (at.front || p.window == 0 || t0 > wp1 - p.window);
    };
    auto unseen_half = [&](const Place &at) {
        const int t0 = at.t0 + kh * 64, end = min(at.last, t0 + 63);
        if constexpr (View::kTexts) return t0 > at.last || (at.text >= 0 && (at.text < first_text || at.text > last_text));
        return t0 > min(wp1, at.last) || (p.window > 0 && !at.front && end <= max(0, wp0) - p.window && t0 >= p.sinks);
    };
    bool skipped = false;

    // ---- one tile: both products and the softmax of this wavefront's 64 keys
    const int v_row = half * 4 + ((lane & 15) >> 2);               // of the first run of four keys; the second one is 8 further
    const int v_piece = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1); // + 4 d
    // fetch_more(ks): f16: called beside every step of the first product (all loads at once hold a wavefront up for 400 cycles); 4 bits: once behind it
    auto work = [&](unsigned stage, int t0, int limit, auto whole, auto fetch_more) __attribute__((always_inline)) {
        const unsigned char *lds_k = lds + stage * kStageBytes + kh * (64 * kRowBytes), *lds_v = lds_k + kTileBytes;
        // S^T: the two 32-key products side by side, K read three steps ahead of them.  (Barriers against reordering: left alone, every read ends up right in
        // front of its product, and its latency in between.)
        float16_t w[2];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int v = 0; v < 16; v++) w[t][v] = 0.0f;
        half8_t k_frag[4][2];
        auto read_k = [&](int ks) {
#pragma unroll
            for (int t = 0; t < 2; t++) k_frag[ks % 4][t] = *reinterpret_cast<const half8_t *>(lds_k + (t * 32 + col) * kRowBytes + (((ks * 2 + half) ^ k_swz(col)) << 4));
        };
        __builtin_amdgcn_s_setprio(1); // a wavefront at its products before one at its softmax (1500 rows with a window: 53.4 -> 50.7 us)
        read_k(0);
        if (kKS > 1) read_k(1);
        if (kKS > 2) read_k(2);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < kKS; ks++) {
            if (ks + 3 < kKS) read_k(ks + 3);
#pragma unroll
            for (int t = 0; t < 2; t++) w[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k_frag[ks % 4][t], q[ks], w[t], 0, 0, 0);
            if constexpr (!kQ4) fetch_more(ks);
            if constexpr (kQ4) { // the next tile's codes are converted beside the products, which leave the vector ALU idle
#pragma unroll
                for (int word = ks * 4 * kItems / kKS; word < (ks + 1) * 4 * kItems / kKS; word++) place_word(1 - stage, word);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        if constexpr (kQ4) fetch_more(0);
        half8_t v_frag[2][kDT];
        auto read_v = [&](int sl, int d) {
            const unsigned char *from = lds_v + (sl * 16 + v_row) * kRowBytes + (((d * 4 + v_piece) ^ v_swz(v_row)) << 4) + (lane & 1) * 8;
            typedef __attribute__((address_space(3))) short4_t *lds4;
            const half4_t a0 = __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(__attribute__((address_space(3))) void *)from));
            const half4_t a1 = __builtin_bit_cast(half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(__attribute__((address_space(3))) void *)(from + 8 * kRowBytes)));
            v_frag[sl & 1][d] = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
        };
#pragma unroll
        for (int d = 0; d < kDT; d++) read_v(0, d);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!decltype(whole)::value) { // a bit per key of the tile (what sees() says of each), and a select by it
            auto ones = [](int n) { return n <= 0 ? 0ull : ~0ull >> (64 - min(n, 64)); };
            const uint64_t seen = (ones(limit - t0 + 1) & (~ones(my_low - t0) | ones(p.sinks - t0))) >> (half * 4);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    const uint32_t all = (uint32_t)((int32_t)((uint32_t)(seen >> (t * 32)) << (31 - (v >> 2) * 8 - (v & 3))) >> 31);
                    w[t][v] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, (float)w[t][v]) & all) | (0xff800000u & ~all)); // else -infinity
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int v = 0; v < 16; v++) top = fmaxf(top, w[t][v]);
        top = fmaxf(top, other_half_lane(top));
        // the reference point follows the maximum when some row's has grown by more than 2^8: weights stay below 2^8 times what they are carried by
        const float m_new = fmaxf(m_run, top);
        if (__any((m_new - m_run) * c2 > 8.0f)) {
            const float alpha = m_run > -INFINITY ? __builtin_amdgcn_exp2f((m_run - m_new) * c2) : 0.0f;
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int d = 0; d < kDT; d++)
#pragma unroll
                for (int v = 0; v < 16; v++) o[d][v] *= alpha;
        }
        const float mc = (m_run > -INFINITY ? m_run * c2 : 0.0f) - kWeightLift;
        // O^T += V^T . W, 16 keys at a time: between the products of one step the weights of the next are formed and its V is read
        half8_t h[2];
        float sum[2] = {0.0f, 0.0f};
        auto weight = [&](int sl, int i) {
            const float e = __builtin_amdgcn_exp2f(fmaf(w[sl / 2][(sl % 2) * 8 + i], c2, -mc));
            sum[i & 1] += e;
            h[sl & 1][i] = (half_t)e;
        };
#pragma unroll
        for (int i = 0; i < 8; i++) weight(0, i);
        __builtin_amdgcn_s_setprio(1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int sl = 0; sl < 4; sl++)
#pragma unroll
            for (int d = 0; d < kDT; d++) {
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v_frag[sl & 1][d], h[sl & 1], o[d], 0, 0, 0);
                if (sl < 3) {
                    read_v(sl + 1, d);
#pragma unroll
                    for (int i = d * 8 / kDT; i < (d + 1) * 8 / kDT; i++) weight(sl + 1, i);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        __builtin_amdgcn_s_setprio(0);
        l_run += sum[0] + sum[1];
    };

    if (kQ4 && tid == 0) sh_wide = 0;
    if (s_first < s_end) {
        Place at = place_of(s_first), ahead = at; // `ahead`: the tile after the one fetched last
        auto fetch_ahead = [&](int s) __attribute__((always_inline)) {
            if (s >= s_end) return;
            fetch(planes_of(ahead), min(kAtKeys, ahead.last - ahead.t0 + 1), (unsigned)(s - s_first) & 1);
            ahead.t0 += kAtKeys;
            ahead.row += kAtKeys;
            if (ahead.t0 > ahead.last) ahead = place_of(s + 1);
        };
        fetch_ahead(s_first);
        place(0);
        if constexpr (kQ4) fetch_ahead(s_first + 1);
        unsigned stage = 0;
        for (int s = s_first; s < s_end; s++) {
            // tiles from here on that every row sees whole and that another tile (f16: a whole one) follows in the same run of rows (wavefronts may count
            // differently: both loops stage and wait alike)
            const int seen = whole_to(at) - kh * 64 - 63 - at.t0, follow = at.last + 1 - at.t0;
            int run = whole_half(at) ? min(min(seen / kAtKeys + 1, (kQ4 ? (follow + kAtKeys - 1) / kAtKeys : follow / kAtKeys) - 1), s_end - 1 - s) : 0;
            if (run > 0) {
                const int end = s + run;
                if constexpr (!kQ4) {
                    ahead.t0 = at.t0 + (run + 1) * kAtKeys;
                    ahead.row = at.row + (run + 1) * kAtKeys;
                    if (ahead.t0 > ahead.last) ahead = place_of(end + 1);
                }
                const PlaneRows planes = planes_of(at);
                size_t row = planes.row + kAtKeys;
                at.t0 += run * kAtKeys;
                at.row += run * kAtKeys;
                do {
                    if constexpr (!kQ4) wait_vmcnt<0>();
                    __syncthreads();
                    work(stage, 0, 0, std::true_type{}, [&](int ks) __attribute__((always_inline)) {
                        if constexpr (kQ4) fetch_ahead(s + 2);
                        else {
                            const half_t *from = reinterpret_cast<const half_t *>(ks < kIssues ? planes.k.data : planes.v.data) + row * HD;
                            const int i = ks % kIssues;
                            dma16_base(from, (unsigned)(my_row + i * kIssueRows) * kRowBytes + (ks < kIssues ? k_from : v_from),
                                       lds_base + (1 - stage) * kStageBytes + (unsigned)(i * kWaves + wave) * 1024u + (ks < kIssues ? 0 : kTileBytes));
                        }
                    });
                    row += kAtKeys;
                    __builtin_amdgcn_sched_barrier(0);
                    stage = 1 - stage;
                } while (++s < end);
            }
            if constexpr (!kQ4) wait_vmcnt<0>(); // this wavefront's part of the tile has landed
            __syncthreads();                     // ... and everybody's; everybody is done with the tile before, whose stage is filled next
            if constexpr (!kQ4) fetch_ahead(s + 1);
            bool use = !unseen_half(at);
            if (use) { // is every value of V finite?
                const unsigned char *v = lds + stage * kStageBytes + kTileBytes + kh * (64 * kRowBytes);
                ushort2_t top = {0, 0};
#pragma unroll 4
                for (int i = 0; i < 64 * kRowBytes / 1024; i++) {
                    const uint4_t x = *reinterpret_cast<const uint4_t *>(v + i * 1024 + lane * 16);
#pragma unroll
                    for (int j = 0; j < 4; j++) top = __builtin_elementwise_max(top, __builtin_bit_cast(ushort2_t, x[j] & 0x7fff7fffu));
                }
                const bool odd = (int)(top[0] >= 0x7c00) | (int)(top[1] >= 0x7c00);
                if (__any(odd) && !whole_half(at)) {
                    skipped = true;
                    use = false;
                }
            }
            if (use) {
                work(stage, at.t0 + kh * 64, limit_of(at), std::false_type{}, [&](int) __attribute__((always_inline)) { if constexpr (kQ4) fetch_ahead(s + 2); });
            } else if constexpr (kQ4) {
                place(1 - stage); // (behind the last tile: into a stage that is read no more)
                fetch_ahead(s + 2);
            }
            __builtin_amdgcn_sched_barrier(0);
            stage = 1 - stage;
            at.t0 += kAtKeys;
            at.row += kAtKeys;
            if (at.t0 > at.last) at = place_of(s + 1);
        }
    }

    bool anew = false; // every tile again
    if constexpr (kQ4) {
        if (wide) sh_wide = 1; // (0 since before the barriers of the loop, without which there is no tile)
        __syncthreads();
        anew = sh_wide != 0;
    }
    if (anew) {
        m_run = -INFINITY;
        l_run = 0.0f;
#pragma unroll
        for (int d = 0; d < kDT; d++)
#pragma unroll
            for (int v = 0; v < 16; v++) o[d][v] = 0.0f;
    }
    if (anew || __any(skipped)) {
        // Tiles that hold a value of V that is not finite and that some row of the wavefront may not see (weight 0 would make a NaN of it in the product)
        // were left out above.  Here every row adds up what it sees, key by key in f32.  So it does with all tiles where 4 bits stand for values that f16
        // does not hold (a group from -65504 to 65504 reads as 65536 at its upper end): 1500 rows of 32 heads on 8 then take 14.6 ms instead of 48 us.
        for (int s = s_first; s < s_end; s++) {
            const Place at = place_of(s);
            if (unseen_half(at) || (!anew && whole_half(at))) continue;
            const int t0 = at.t0 + kh * 64, here = min(64, at.last - t0 + 1), limit = limit_of(at);
            const PlaneRows planes = planes_of(at);
            const size_t row = planes.row + kh * 64;
            if (!anew) {
                bool odd = false;
                for (int i = lane; i < here * HD; i += 64) odd |= !(fabsf(plane_load1<CT>(planes.v, row * HD + i)) < INFINITY);
                if (!__any(odd)) continue;
            }
#pragma unroll 1
            for (int j = 0; j < here; j++) {
                const size_t from = (row + j) * HD;
                float dot = 0.0f;
#pragma unroll 1
                for (int d = half * (HD / 2); d < (half + 1) * (HD / 2); d++) dot = fmaf((float)q_row[d], plane_load1<CT>(planes.k, from + d), dot);
                dot += __shfl_xor(dot, 32, 64);
                const bool seen = sees(t0 + j, limit);
                const float m_new = seen ? fmaxf(m_run, dot) : m_run;
                const float alpha = m_new > -INFINITY ? __builtin_amdgcn_exp2f((m_run - m_new) * c2) : 1.0f;
                const float wt = seen ? __builtin_amdgcn_exp2f(fmaf(dot - (m_new > -INFINITY ? m_new : 0.0f), c2, kWeightLift)) : 0.0f;
                m_run = m_new;
                l_run = fmaf(l_run, alpha, half == 0 ? wt : 0.0f);
#pragma unroll
                for (int d = 0; d < kDT; d++)
#pragma unroll
                    for (int v = 0; v < 16; v++) {
                        const int dim8 = (v >> 2) * 8, in8 = half * 4 + (v & 3); // place in O^T
                        const float x = plane_load1<CT>(planes.v, from + d * 32 + dim8 + (kQ4 ? (in8 >> 1) + 4 * (in8 & 1) : in8));
                        o[d][v] = seen ? fmaf(wt, x, o[d][v] * alpha) : o[d][v];
                    }
            }
        }
    }

    __syncthreads(); // everybody is done with the tiles
    if constexpr (kShares > 1) { // the second half of the keys hands its (O, m, sum) to the first
        float *join = reinterpret_cast<float *>(lds) + rg * kJoinFloats + lane;
        if (kh == 1) {
#pragma unroll
            for (int d = 0; d < kDT; d++)
#pragma unroll
                for (int v = 0; v < 16; v++) join[(d * 16 + v) * 64] = o[d][v];
            join[(kDT * 16) * 64] = m_run;
            join[(kDT * 16 + 1) * 64] = l_run;
        }
        __syncthreads();
        if (kh == 1) return;
        const float m1 = join[(kDT * 16) * 64], l1 = join[(kDT * 16 + 1) * 64], m = fmaxf(m_run, m1);
        const float a0 = m_run > -INFINITY ? __builtin_amdgcn_exp2f((m_run - m) * c2) : 0.0f, a1 = m1 > -INFINITY ? __builtin_amdgcn_exp2f((m1 - m) * c2) : 0.0f;
        l_run = (m_run > -INFINITY ? l_run * a0 : l_run) + (m1 > -INFINITY ? l1 * a1 : l1); // (nothing seen: 0; only NaN: NaN)
        m_run = m;
#pragma unroll
        for (int d = 0; d < kDT; d++)
#pragma unroll
            for (int v = 0; v < 16; v++) {
                const float x = join[(d * 16 + v) * 64];
                o[d][v] = (a0 > 0.0f ? o[d][v] * a0 : 0.0f) + (a1 > 0.0f ? x * a1 : 0.0f);
            }
    }
    const float l = my_p < 0 ? 0.0f : l_run + __shfl_xor(l_run, 32, 64); // (padding: 0)
    if (kShares > 1 && (v.partial() || n_pieces > 1)) { // ---- leave (m, sum) and O of the piece for the join
        if (w0 + col > r1) return;
        float *ws = v.partials(unit, rows, w0 + col, HD);
        const int slot = v.first_slot + piece;
        if (half == 0) {
            ws[2 * slot] = m_run;
            ws[2 * slot + 1] = l;
        }
        ws += 2 * v.pieces + (size_t)slot * HD;
#pragma unroll
        for (int d = 0; d < kDT; d++)
#pragma unroll
            for (int x = 0; x < 4; x++) {
                float *to = ws + d * 32 + x * 8;
                if constexpr (kQ4) { // places 4 half + i of eight hold dims (place / 2) + 4 (place % 2)
                    *reinterpret_cast<float2 *>(to + 2 * half) = make_float2(o[d][x * 4], o[d][x * 4 + 2]);
                    *reinterpret_cast<float2 *>(to + 2 * half + 4) = make_float2(o[d][x * 4 + 1], o[d][x * 4 + 3]);
                } else {
                    *reinterpret_cast<float2 *>(to + 4 * half) = make_float2(o[d][x * 4], o[d][x * 4 + 1]);
                    *reinterpret_cast<float2 *>(to + 4 * half + 2) = make_float2(o[d][x * 4 + 2], o[d][x * 4 + 3]);
                }
            }
        return;
    }
    // ---- normalise, round to f16, turn O^T into rows through LDS and store 16-byte pieces
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    half_t *ot = reinterpret_cast<half_t *>(lds + rg * (kShares > 1 ? kJoinFloats * 4 : 32 * kOutRow * 2));
#pragma unroll
    for (int d = 0; d < kDT; d++)
#pragma unroll
        for (int x = 0; x < 4; x++) {
            half4_t y;
#pragma unroll
            for (int i = 0; i < 4; i++) y[i] = (half_t)(l == 0.0f ? 0.0f : o[d][x * 4 + i] * inv);
            half_t *to = ot + col * kOutRow + d * 32 + x * 8;
            if constexpr (kQ4) { // (as above)
                *reinterpret_cast<half2_t *>(to + 2 * half) = half2_t{y[0], y[2]};
                *reinterpret_cast<half2_t *>(to + 2 * half + 4) = half2_t{y[1], y[3]};
            } else {
                *reinterpret_cast<half4_t *>(to + 4 * half) = y;
            }
        }
    // (a wavefront reads back only what it wrote)
    half_t *out = reinterpret_cast<half_t *>(p.out);
#pragma unroll
    for (int i = 0; i < 32 * kPieces / 64; i++) {
        const int at = i * 64 + lane, r = w0 + at / kPieces, c = at % kPieces;
        if (r > r1) continue;
        const int ri = r / group;
        *reinterpret_cast<half8_t *>(out + ((size_t)(b * p.n + ri) * p.n_heads + g * group + (r - ri * group)) * HD + c * 8) =
            *reinterpret_cast<const half8_t *>(ot + (at / kPieces) * kOutRow + c * 8);
    }
}

} // namespace rlh
