// attn_shared.hip -- attention of a batch of texts that share a long prefix.
//
// The row at own position p of text b sees the prefix's positions 0 .. P - 1 and the text's 0 .. p:
//   out = (sum over both of w_t v_t) / (sum of w_t),  w_t = exp(q . k_t / sqrt(hd) - m).
// Sums over parts of the positions, each with a reference point m of its own, join into one: so the prefix is read once for the rows of all texts that share a key and value
// head, instead of once per text.
//
// A workgroup takes rows of one key and value head, whatever texts they are of; its steps are the prefix's and then every one of its texts', masked for the rows of the others.  They
// are cut into pieces; where there is only one the result is final, and pieces leave (m, sum, O) of their rows in work memory, which a second launch joins.
//   Few rows or few positions, f32 arithmetic, or where nothing may be rounded but the result: 16 rows at a time, from memory into registers (attn_rows_device.h).
//   Many rows of each text and many positions: 128 rows at a time, through tiles of keys in LDS (attn_tiles_device.h, f16 arithmetic).
//   Many rows and positions, but few rows of each text: the prefix in tiles; 128 rows would be of too many texts for the texts' own positions, which go 16 rows at a time beside them in the same launch.
//
// Measured (heads of 128): a row each of 4 texts behind 383 positions, 32 heads: 9.8 us, the latency of one workgroup per head; of 64 texts behind 6001, 32 heads on 8: 26 us, 60 MB; of
// 16 texts behind 65700, 64 heads on 8, 4 bits: 58 us, 590 TFLOP/s, conversions beside the products; 3 rows of 8 texts behind 1031, 32 heads in f32: 20 us, 2.3 TB/s of memory;
// 61 rows of 16 texts behind 2107, 40 heads: 78 us, 545 TFLOP/s.  A launch that joins pieces: 3 to 5 us of those.
#include "kernels.h"
#include "answers.h"
#include "attn_rows_device.h"
#include "attn_tiles_device.h"

#include <algorithm>

namespace rlh {

struct SharedKernelParams {
    AttnSharedParams a;
    float *ws; // for every row, from `cut` on, of every key and value head the pairs (m, sum) of all its pieces, then the sums O of each
    int slots; // places for pieces
    int cut;
    SharedPart part[2]; // in tiles; 16 rows at a time
};

constexpr int kMaxTexts = 16; // of a workgroup; a row of lanes
// The steps of a workgroup: the prefix's, and every one of its texts' own.
template <int kStep>
struct TextsWalk {
    int steps, prefix_steps, prefix_last;
    int first_text, first, last; // of lane l: the first step and the last position of text first_text + l
    struct At {
        int t0, last, text;
    };
    __device__ At at(int s) const {
        if (s < prefix_steps) return At{s * kStep, prefix_last, -1};
        const int l = 63 - __builtin_clzll(__ballot(first <= s)); // (texts without a step start where the next one does)
        return At{(s - __builtin_amdgcn_readlane(first, l)) * kStep, __builtin_amdgcn_readlane(last, l), first_text + l};
    }
};

// A part as the kernels see it.
struct PartParams {
    static constexpr int window = 0, sinks = 0;
    const void *q;
    void *out;
    int n_heads, n_kv, max_seq_len, n;
};
// Rows of all texts, row i is row i % n of text i / n.
struct SharedView {
    PartParams p;
    const AttnSharedParams &a;
    float *const &ws; // (references, as in WindowView)
    const int &pieces, &first_slot, &cut;
    int piece_steps;
    __device__ SharedView(const SharedKernelParams &c, int part, bool whole)
        : p{c.a.q, c.a.out, c.a.n_heads, c.a.n_kv, c.a.prefix_rows, c.a.n * c.a.n_seqs}, a(c.a), ws(c.ws), pieces(c.slots), first_slot(c.part[part].first_slot), cut(c.cut),
          piece_steps(whole ? 1 << 30 : c.part[part].piece_steps) {}
    __device__ float *partials(int g, int rows, int r, int hd) const { return ws + ((size_t)g * (rows - cut) + r - cut) * pieces * (hd + 2); }
};
// The prefix alone: all rows are at its last position, padding too, and a join tells these apart.  (There is always one: of a call that sees a prefix some row has a position
// of its own, so the texts' part has a piece.)
struct PrefixView : SharedView {
    static constexpr bool kTexts = false;
    __device__ explicit PrefixView(const SharedKernelParams &c) : SharedView(c, 0, false) {}
    __device__ constexpr bool partial() const { return true; }
    __device__ int start(int) const { return a.prefix_len - 1; }
    __device__ int position(int start, int) const { return start; }
    __device__ int text(int) const { return 0; }
    __device__ PlaneRows planes(int g, int, int row) const { return {a.prefix_k, a.prefix_v, (size_t)g * a.prefix_rows + row}; }
};
// The texts' own positions, kPrefix: behind the prefix.
template <bool kPrefix>
struct TextsView : SharedView {
    static constexpr bool kTexts = true;
    __device__ TextsView(const SharedKernelParams &c, int part, bool whole) : SharedView(c, part, whole) {}
    __device__ constexpr bool partial() const { return !kPrefix; }
    __device__ int start(int) const { return 0; }
    __device__ int text(int i) const { return i / a.n; }
    __device__ int position(int, int i) const { return a.start[i / a.n] + i % a.n; }
    __device__ PlaneRows planes(int g, int text, int row) const {
        if (kPrefix && text < 0) return {a.prefix_k, a.prefix_v, (size_t)g * a.prefix_rows + row};
        return {a.cache_k, a.cache_v, ((size_t)text * a.n_kv + g) * a.max_seq_len + row};
    }
    template <int kStep>
    __device__ TextsWalk<kStep> walk(int r0, int r1, int lane) const {
        const int group = a.n_heads / a.n_kv, rows = a.n * group;
        TextsWalk<kStep> w;
        w.prefix_last = a.prefix_len - 1;
        w.prefix_steps = kPrefix ? (a.prefix_len + kStep - 1) / kStep : 0;
        w.first_text = r0 / rows;
        const int text = w.first_text + lane; // (16 of them at most: 16 rows, or 128 of more than 32 for each)
        w.last = text <= r1 / rows ? a.start[min(text, a.n_seqs - 1)] + (min(r1, (text + 1) * rows - 1) - text * rows) / group : -1;
        const int mine = w.last < 0 ? 0 : w.last / kStep + 1;
        int sum = mine; // of the lanes up to this one
        sum += __builtin_amdgcn_update_dpp(0, sum, 0x111, 0xf, 0xf, true); // (row_shr: from so many lanes below)
        sum += __builtin_amdgcn_update_dpp(0, sum, 0x112, 0xf, 0xf, true);
        sum += __builtin_amdgcn_update_dpp(0, sum, 0x114, 0xf, 0xf, true);
        sum += __builtin_amdgcn_update_dpp(0, sum, 0x118, 0xf, 0xf, true);
        w.first = lane < kMaxTexts ? w.prefix_steps + sum - mine : INT32_MAX;
        w.steps = w.prefix_steps + __builtin_amdgcn_readlane(sum, kMaxTexts - 1);
        return w;
    }
};

// kForm: what goes through tiles.  (LDS for them leaves room for one workgroup per compute unit.)
enum SharedForm { kNoTiles, kPrefixTiles, kAllTiles };
template <typename AC, typename QT, typename CT, int HD, int kForm>
__global__ __launch_bounds__(kAwThreads, kForm == kNoTiles ? 1 : 2) void attn_shared_kernel(SharedKernelParams c) {
    constexpr int kTilesBytes = kForm == kNoTiles ? 0 : TilesShared<HD, 2>::kBytes, kRowsBytes = kForm == kAllTiles ? 0 : (int)sizeof(RowsShared<HD>);
    __shared__ __attribute__((aligned(1024))) unsigned char lds[kTilesBytes > kRowsBytes ? kTilesBytes : kRowsBytes];
    __shared__ int wide;
    // tiles first; those of one stretch of keys are a multiple of the number of heads apart, on one XCD where that is a multiple of eight
    int at = blockIdx.x;
    const int first = kForm == kNoTiles ? 0 : c.a.n_kv * c.part[0].blocks * c.part[0].pieces, own = kForm == kNoTiles || (kForm == kPrefixTiles && at >= first) ? 1 : 0;
    if (own) at -= first;
    // blocks that are not cut, and then the pieces of the others
    const int g = at % c.a.n_kv, rest = at / c.a.n_kv, uncut = c.part[own].whole, cut = c.part[own].blocks - uncut;
    const bool whole = rest < uncut;
    const int block = whole ? rest : uncut + (rest - uncut) % cut, piece = whole ? 0 : (rest - uncut) / cut;
    if constexpr (kForm == kNoTiles) {
        attn_rows<AC, QT, CT, HD>(TextsView<true>(c, 1, whole), *reinterpret_cast<RowsShared<HD> *>(lds), g, block, piece);
    } else if constexpr (kForm == kAllTiles) {
        attn_tiles<CT, HD, 2>(TextsView<true>(c, 0, whole), lds, wide, g, block, piece);
    } else {
        if (own) attn_rows<AC, QT, CT, HD>(TextsView<false>(c, 1, false), *reinterpret_cast<RowsShared<HD> *>(lds), g, block, piece);
        else attn_tiles<CT, HD, 2>(PrefixView(c), lds, wide, g, block, piece);
    }
}

constexpr int kSharedTile = 128; // positions of a step in tiles
// Where row r of a key and value head's is, and how many pieces it has.
struct JoinRow {
    int n_pieces;
    bool padding, finished;
    size_t out;
    __device__ JoinRow(const SharedKernelParams &c, int g, int r, int hd, int step) { // step: positions, of 16 rows at a time
        const AttnSharedParams &a = c.a;
        const int group = a.n_heads / a.n_kv, rows = a.n * group, b = r / rows, own = r - b * rows, i = own / group, start = a.start[b];
        padding = start + i < 0;
        out = ((size_t)(b * a.n + i) * a.n_heads + g * group + (own - i * group)) * hd;
        const bool in_tiles = c.part[0].texts;
        const SharedPart &part = c.part[in_tiles ? 0 : 1];
        const int together = in_tiles ? kAtRows : kAwRows, r0 = r / together * together, r1 = min(a.n_seqs * rows, r0 + together) - 1;
        if (in_tiles) step = kSharedTile;
        int steps = part.prefix ? (a.prefix_len + step - 1) / step : 0;
        for (int t = r0 / rows; t <= r1 / rows; t++) {
            const int last = a.start[t] + (min(r1, (t + 1) * rows - 1) - t * rows) / group;
            steps += last < 0 ? 0 : last / step + 1;
        }
        n_pieces = (steps + part.piece_steps - 1) / part.piece_steps;
        finished = n_pieces <= 1 && part.prefix;
        if (!part.prefix) n_pieces += c.part[0].pieces;
    }
};

// The rows that were cut join their pieces: a workgroup for a row, where there are few.
template <typename QT, int HD, int kRowsStep>
__global__ __launch_bounds__(kAjWaves *kWave) void attn_shared_join_kernel(SharedKernelParams c) {
    __shared__ float part[kAjWaves * (kWave / (HD / 2))][HD];
    const int g = blockIdx.y, r = c.cut + blockIdx.x, all = gridDim.x;
    const JoinRow row(c, g, r, HD, kRowsStep);
    QT *out = reinterpret_cast<QT *>(c.a.out) + row.out;
    if (row.finished) return;
    if (row.padding) {
        if ((int)threadIdx.x < HD) out[threadIdx.x] = (QT)0.0f;
        return;
    }
    join_pieces<QT, HD, kAjWaves>(part, c.ws + ((size_t)g * all + blockIdx.x) * c.slots * (HD + 2), c.slots, row.n_pieces, [&] { return out; });
}

// ... HD / 4 lanes for a row, where there are many: every lane works out the pieces' weights for itself, eight pieces at a time with a running reference point, and adds up four
// dims.  (39040 rows of two pieces: 21 us with a wavefront for each and its sums through LDS.)
template <typename QT, int HD, int kRowsStep>
__global__ __launch_bounds__(256) void attn_shared_join_rows_kernel(SharedKernelParams c, int all) {
    constexpr int kLanes = HD / 4, kRows = 256 / kLanes, kBatch = 4;
    const int g = blockIdx.y, at = blockIdx.x * kRows + (int)threadIdx.x / kLanes, r = c.cut + at, d = ((int)threadIdx.x % kLanes) * 4;
    if (at >= all) return;
    const JoinRow row(c, g, r, HD, kRowsStep);
    if (row.finished) return;
    const float *ws = c.ws + ((size_t)g * all + at) * c.slots * (HD + 2);
    const float c2 = 1.44269504088896340736f / sqrtf((float)HD);
    float M = -INFINITY, L = 0.0f;
    float4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < (row.padding ? 0 : row.n_pieces); s0 += kBatch) {
        float2 ml[kBatch];
        float2 x[kBatch][2];
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
            const int s = min(s0 + u, row.n_pieces - 1);
            ml[u] = *reinterpret_cast<const float2 *>(ws + 2 * s);
            x[u][0] = *reinterpret_cast<const float2 *>(ws + 2 * c.slots + (size_t)s * HD + d);
            x[u][1] = *reinterpret_cast<const float2 *>(ws + 2 * c.slots + (size_t)s * HD + d + 2);
        }
        float top = M;
#pragma unroll
        for (int u = 0; u < kBatch; u++)
            if (s0 + u < row.n_pieces) top = fmaxf(top, ml[u].x);
        const float before = M > -INFINITY ? __builtin_amdgcn_exp2f((M - top) * c2) : 0.0f;
        M = top;
        L = before > 0.0f ? L * before : L; // (only NaN so far: NaN)
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = before > 0.0f ? o[e] * before : 0.0f;
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
            if (s0 + u >= row.n_pieces) continue;
            const float f = ml[u].x > -INFINITY ? __builtin_amdgcn_exp2f((ml[u].x - M) * c2) : 0.0f;
            L += ml[u].x > -INFINITY ? ml[u].y * f : ml[u].y;
            if (f > 0.0f) {
                o[0] = fmaf(x[u][0].x, f, o[0]);
                o[1] = fmaf(x[u][0].y, f, o[1]);
                o[2] = fmaf(x[u][1].x, f, o[2]);
                o[3] = fmaf(x[u][1].y, f, o[3]);
            }
        }
    }
    QT *out = reinterpret_cast<QT *>(c.a.out) + row.out + d;
    typedef QT vec __attribute__((ext_vector_type(4)));
    vec y;
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = (QT)(L == 0.0f ? 0.0f : o[e] / L);
    *reinterpret_cast<vec *>(out) = y;
}

static bool f16_arithmetic(const AttnSharedParams &p) { return p.f16 && p.cache != kPlaneF32; }

// When `count[k]` workgroups of us[k] each, the first kind first, end on so many places.
static double makespan(int places, const int64_t (&count)[2], const double (&us)[2]) {
    const int64_t whole = count[0] / places, extra = count[0] % places; // `extra` places have one more
    const double busy[2] = {(double)(whole + 1) * us[0], (double)whole * us[0]};
    const double first = count[0] > 0 ? busy[extra > 0 ? 0 : 1] : 0.0;
    if (count[1] == 0) return first;
    const int64_t n[2] = {extra, places - extra};
    const double mean = (busy[0] * (double)n[0] + busy[1] * (double)n[1] + us[1] * (double)count[1]) / places;
    double end = std::max(mean, busy[1] + us[1]);
    const double per_us = 1.0 / us[1];
    for (int tries = 0; tries < 8; tries++, end += 0.25 * us[1]) { // (each leaves room for a quarter of a workgroup more on every place)
        int64_t room = 0;
        for (int k = 0; k < 2; k++)
            if (end > busy[k]) room += n[k] * (int)((end - busy[k]) * per_us + 1e-9);
        if (room >= count[1]) break;
    }
    return std::max(end, first);
}

// How a call is cut, with or without tiles, and how long that takes.  A workgroup of 16 rows takes `fixed` and `per_step` for every step (32 positions, 16 in f32) of its busiest wavefront;
// one of 128 rows the same for every 128 positions; partial results go to memory and back, and a launch joins them.  The numbers of pieces with the least sum are taken.
// The tiles' workgroups start first, the others fill what is left.
static double plan_form(const AttnSharedParams &a, int compute_units, bool tiles, SharedPlan &c) {
    c = SharedPlan{};
    const int group = a.n_heads / a.n_kv;
    const int64_t rows = (int64_t)a.n * group, all = rows * a.n_seqs;
    const bool f16 = f16_arithmetic(a), q4 = a.cache == kPlaneQ4;
    const double size = a.head_dim / 128.0;
    const double launch = tiles ? 0.0 : 2.0, fixed[2] = {7.0, tiles ? 3.0 : 2.0}, per_step[2] = {(q4 ? 2.6 : 1.9) * size, tiles ? (q4 ? 1.6 : 1.2) * size : (q4 ? 1.15 : 1.0) * (0.6 + 1.4 * size)};
    const int step[2] = {kSharedTile, f16 ? 32 : 16}, together[2] = {kAtRows, kAwRows};
    // which parts there are, and what they have
    const bool texts_tiles = tiles && (rows > 2 * kAwRows || a.prefix_len == 0);
    c.part[0].prefix = tiles;
    c.part[0].texts = texts_tiles;
    c.part[1].prefix = !tiles;
    c.part[1].texts = !texts_tiles;
    int longest[2] = {0, 0}; // steps of a workgroup
    double mean[2] = {0.0, 0.0};
    for (int k = 0; k < 2; k++) {
        SharedPart &p = c.part[k];
        if (!p.prefix && !p.texts) continue;
        p.blocks = (int)((all + together[k] - 1) / together[k]);
        const int first = p.prefix ? (a.prefix_len + step[k] - 1) / step[k] : 0;
        longest[k] = first;
        mean[k] = first;
        for (int t = 0; p.texts && t < p.blocks; t++) {
            const int64_t r0 = (int64_t)t * together[k], r1 = std::min(all, r0 + together[k]) - 1;
            int steps = first;
            for (int64_t b = r0 / rows; b <= r1 / rows; b++) {
                const int64_t last = a.start[b] + (std::min(r1, (b + 1) * rows - 1) - b * rows) / group;
                steps += last < 0 ? 0 : (int)(last / step[k]) + 1;
            }
            longest[k] = std::max(longest[k], steps);
            mean[k] += (double)(steps - first) / p.blocks;
        }
    }
    const int places = compute_units; // (small workgroups that share one take turns)
    const int most[2] = {std::min(kMaxPieces / 2, longest[0]), std::min(kMaxPieces / 2, (longest[1] + kAwWaves - 1) / kAwWaves)};
    auto time_of = [&](int k, int n) { // a workgroup of average length, cut into n
        const double part = n > 0 ? std::min((double)((longest[k] + n - 1) / n), mean[k]) : 0.0;
        return fixed[k] + (k ? (double)(((int64_t)part + kAwWaves - 1) / kAwWaves) : part) * per_step[k];
    };
    auto join_time = [&](int64_t rows, int n) { return 3.0 + (double)rows * a.n_kv * n * (a.head_dim + 2) * 8 / 4.5e6; };
    double least = -1.0;
    int pieces[2] = {0, 0};
    if (c.part[0].texts || c.part[1].prefix) { // one part
        const int k = c.part[0].texts ? 0 : 1;
        SharedPart &p = c.part[k];
        // Cut all blocks, or what is left behind as many whole ones as there is room for at a time (16 questions of 61 tokens on 40 heads, 320 blocks for 256 places: 85 -> 78 us)
        const int rounds = (int)((int64_t)a.n_kv * p.blocks / places * places / a.n_kv), whole[2] = {0, rounds < p.blocks ? rounds : 0};
        for (int n = std::min(1, most[k]); n <= most[k]; n += 1 + n / 4) {
            for (int w = 0; w < (whole[1] > 0 && n > 1 ? 2 : 1); w++) {
                const int64_t count[2] = {(int64_t)a.n_kv * whole[w], (int64_t)a.n_kv * (p.blocks - whole[w]) * n};
                const double us[2] = {time_of(k, 1), time_of(k, n)};
                const double end = makespan(places, count, us) + (n > 1 ? join_time(all - (int64_t)whole[w] * together[k], n) : 0.0);
                if (least < 0.0 || end < least) {
                    least = end;
                    pieces[k] = n;
                    p.whole = whole[w];
                }
            }
            if (most[k] == 0) break;
        }
        if (pieces[k] > 1) c.cut = p.whole * together[k];
    } else {
        for (int n0 = 1; n0 <= most[0]; n0 += 1 + n0 / 4) {
            for (int n1 = std::min(1, most[1]); n1 <= most[1]; n1 += 1 + n1 / 4) {
                const int64_t count[2] = {(int64_t)a.n_kv * c.part[0].blocks * n0, (int64_t)a.n_kv * c.part[1].blocks * n1};
                const double us[2] = {time_of(0, n0), time_of(1, n1)};
                const double end = makespan(places, count, us) + (n0 + n1 > 1 ? join_time(all, n0 + n1) : 0.0);
                if (least < 0.0 || end < least) {
                    least = end;
                    pieces[0] = n0;
                    pieces[1] = n1;
                }
                if (most[1] == 0) break;
            }
        }
    }
    for (int k = 0; k < 2; k++) {
        SharedPart &p = c.part[k];
        p.piece_steps = pieces[k] > 0 ? (longest[k] + pieces[k] - 1) / pieces[k] : 1;
        if (k && pieces[k] > 1) p.piece_steps = (p.piece_steps + kAwWaves - 1) / kAwWaves * kAwWaves; // (a step for every wavefront: eight texts' drafts in f32 22.7 -> 21.2 us)
        p.pieces = (longest[k] + p.piece_steps - 1) / p.piece_steps;
        if (p.prefix && p.texts) p.pieces = std::max(1, p.pieces); // (nothing but padding: zeros)
        p.first_slot = k ? c.part[0].pieces : 0;
        c.slots += p.pieces;
        c.workgroups += (int64_t)a.n_kv * (p.whole + (p.blocks - p.whole) * (int64_t)p.pieces);
    }
    c.joined = c.slots > 1;
    c.work_floats = c.joined ? (size_t)(all - c.cut) * a.n_kv * c.slots * (a.head_dim + 2) : 0;
    return least + launch;
}
SharedPlan plan_attn_shared(const AttnSharedParams &a, int compute_units) {
    const int64_t rows = (int64_t)a.n * (a.n_heads / a.n_kv), all = rows * a.n_seqs;
    SharedPlan c, d;
    const double us = plan_form(a, compute_units, false, c);
    // Tiles take 128 rows of one head, of up to 16 texts where these go through tiles as well.  The estimates cost nothing over the faster form on average over 180 calls of all sizes, 23 % at
    // worst; tiles for all of more than 32 rows took up to 2.5 times as long (245 rows of 16 heads behind 120 positions 20 us, 8; 1722 rows of 4 heads behind 8316 are 49 in tiles and 151).
    // Working this out takes 0.04 to 4 us of host time for up to 256 texts of 8 rows, 36 for 131072 rows of a key and value head.
    if (a.form == 1 || !f16_arithmetic(a) || a.exact || all <= 2 * kAwRows || (a.prefix_len == 0 && rows < kAtRows / (kMaxTexts - 1) + 1)) return c;
    return plan_form(a, compute_units, true, d) < us || a.form == 2 ? d : c;
}

template <typename AC, typename QT, typename CT, int HD>
static void launch_shared(const SharedKernelParams &c, const SharedPlan &plan, hipStream_t s) {
    const dim3 grid((unsigned)plan.workgroups), block(kAwThreads);
    if constexpr (std::is_same_v<AC, half_t>) {
        if (c.part[0].texts) hipLaunchKernelGGL((attn_shared_kernel<AC, QT, CT, HD, kAllTiles>), grid, block, 0, s, c);
        else if (c.part[0].prefix) hipLaunchKernelGGL((attn_shared_kernel<AC, QT, CT, HD, kPrefixTiles>), grid, block, 0, s, c);
    }
    if (!c.part[0].prefix) hipLaunchKernelGGL((attn_shared_kernel<AC, QT, CT, HD, kNoTiles>), grid, block, 0, s, c);
    if (!plan.joined) return;
    const unsigned rows = (unsigned)(c.a.n * c.a.n_seqs * (c.a.n_heads / c.a.n_kv) - c.cut), per = 256 / (HD / 4);
    constexpr int kStep = Step<AC, CT, HD>::kPositions;
    if ((int64_t)rows * c.a.n_kv <= 1024) hipLaunchKernelGGL((attn_shared_join_kernel<QT, HD, kStep>), dim3(rows, (unsigned)c.a.n_kv), dim3(kAjWaves * kWave), 0, s, c);
    else hipLaunchKernelGGL((attn_shared_join_rows_kernel<QT, HD, kStep>), dim3((rows + per - 1) / per, (unsigned)c.a.n_kv), dim3(256), 0, s, c, (int)rows);
}
template <typename AC, typename QT, typename CT>
static hipError_t launch_hd(const SharedKernelParams &c, const SharedPlan &plan, hipStream_t s) {
    switch (c.a.head_dim) {
    case 32: launch_shared<AC, QT, CT, 32>(c, plan, s); break;
    case 64: launch_shared<AC, QT, CT, 64>(c, plan, s); break;
    case 128: launch_shared<AC, QT, CT, 128>(c, plan, s); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_attn_shared(const AttnSharedParams &a, const SharedPlan &plan, float *ws, hipStream_t s) {
    SharedKernelParams c{a, ws, plan.slots, plan.cut, {plan.part[0], plan.part[1]}};
    switch (a.cache * 2 + a.f16) {
    case kPlaneF16 * 2: return launch_hd<float, float, half_t>(c, plan, s);
    case kPlaneF16 * 2 + 1: return launch_hd<half_t, half_t, half_t>(c, plan, s);
    case kPlaneF32 * 2: return launch_hd<float, float, float>(c, plan, s);
    case kPlaneF32 * 2 + 1: return launch_hd<float, half_t, float>(c, plan, s);
    case kPlaneQ4 * 2: return launch_hd<float, float, Quant4>(c, plan, s);
    case kPlaneQ4 * 2 + 1: return launch_hd<half_t, half_t, Quant4>(c, plan, s);
    default: return hipErrorInvalidValue;
    }
}

} // namespace rlh
