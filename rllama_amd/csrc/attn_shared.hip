// attn_shared.hip -- attention of a batch of texts that share a long prefix.
//
// The row at own position p of text b sees the prefix's positions 0 .. P - 1 and the text's 0 .. p:
//   out = (sum over both of w_t v_t) / (sum of w_t),  w_t = exp(q . k_t / sqrt(hd) - m).
// Sums over parts of the positions, each with a reference point m of its own, join into one: so the prefix is read once for the rows of all texts that share a key and value
// head, instead of once per text.
//
// Few rows per key and value head, or f32 arithmetic: 16 rows at a time, whatever texts they are of, from memory into registers (attn_rows_device.h).  A tile's steps are the prefix's and
// then every one of its texts', masked for the rows of the others; they are cut into pieces, and where there is only one the result is final.
// Many: the prefix through tiles of keys in LDS for 128 rows (attn_tiles_device.h, f16 arithmetic), and the texts' own positions beside it in the same launch: 16 rows at a time as above, or,
// where a text alone has many rows, in tiles as well.  Pieces leave (m, sum, O) of their rows in work memory, and a second launch joins them.
#include "kernels.h"
#include "answers.h"
#include "attn_rows_device.h"
#include "attn_tiles_device.h"

#include <algorithm>

namespace rlh {

struct SharedKernelParams {
    AttnSharedParams a;
    float *ws; // for every row of every key and value head the pairs (m, sum) of all its pieces, then the sums O of each
    int slots; // places for pieces
    SharedPart part[2]; // the prefix in tiles (none where everything goes 16 rows at a time); the rest
};

// The steps of a tile of 16 rows: the prefix's, and every text's own.
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
    PlaneRef cache_k, cache_v;
    int n_heads, n_kv, max_seq_len, n;
};
struct SharedView {
    PartParams p;
    const AttnSharedParams &a;
    int own; // 0: the prefix in tiles, 1: the rest
    int prefix_len; // of the rest
    float *ws;
    int pieces, piece_steps, first_slot;
    bool apart; // results are left for a join whatever the number of pieces
    // rows of one text of the unit (texts in tiles), or of all (the prefix, and 16 rows at a time)
    __device__ SharedView(const SharedKernelParams &c, int part, bool one_text)
        : p{c.a.q, c.a.out, part ? c.a.cache_k : c.a.prefix_k, part ? c.a.cache_v : c.a.prefix_v, c.a.n_heads, c.a.n_kv, part ? c.a.max_seq_len : c.a.prefix_rows,
            one_text ? c.a.n : c.a.n * c.a.n_seqs},
          a(c.a), own(part), prefix_len(c.part[0].pieces > 0 ? 0 : c.a.prefix_len), ws(c.ws), pieces(c.slots), piece_steps(c.part[part].piece_steps), first_slot(c.part[part].first_slot),
          apart(c.part[0].pieces > 0 || c.part[1].tiles) {}
    __device__ bool partial() const { return apart; }
    __device__ float *partials(int unit, int rows, int r, int hd) const { // a row's place among those of all texts
        const int b = unit / a.n_kv, g = unit - b * a.n_kv;
        return ws + ((size_t)g * (a.n_seqs * a.n * (a.n_heads / a.n_kv)) + (size_t)b * rows + r) * pieces * (hd + 2);
    }
};
// tiles: all rows of the prefix's part are at its last position
struct TilesView : SharedView {
    __device__ TilesView(const SharedKernelParams &c, int part) : SharedView(c, part, part == 1) {}
    __device__ int start(int b) const { return own ? a.start[b] : a.prefix_len - 1; }
    __device__ int position(int start, int i) const { return own ? start + i : start; }
};
// 16 rows of all texts at a time: row i is row i % n of text i / n
struct TextsView : SharedView {
    static constexpr bool kTexts = true;
    __device__ explicit TextsView(const SharedKernelParams &c) : SharedView(c, 1, false) {}
    __device__ int start(int) const { return 0; }
    __device__ int text(int i) const { return i / a.n; }
    __device__ int position(int, int i) const { return a.start[i / a.n] + i % a.n; }
    __device__ PlaneRows planes(int text, int g, int row) const {
        if (text < 0) return {a.prefix_k, a.prefix_v, (size_t)g * a.prefix_rows + row};
        return {a.cache_k, a.cache_v, ((size_t)text * a.n_kv + g) * a.max_seq_len + row};
    }
    template <int kStep>
    __device__ TextsWalk<kStep> walk(int r0, int r1, int lane) const {
        const int group = a.n_heads / a.n_kv, rows = a.n * group;
        TextsWalk<kStep> w;
        w.prefix_last = prefix_len - 1;
        w.prefix_steps = (prefix_len + kStep - 1) / kStep;
        w.first_text = r0 / rows;
        const int text = w.first_text + lane; // (16 of them at most)
        w.last = text <= r1 / rows ? a.start[min(text, a.n_seqs - 1)] + (min(r1, (text + 1) * rows - 1) - text * rows) / group : -1;
        const int mine = w.last < 0 ? 0 : w.last / kStep + 1;
        int sum = mine;
#pragma unroll
        for (int off = 1; off < kAwRows; off <<= 1) {
            const int up = __shfl_up(sum, off, kWave);
            if (lane >= off) sum += up;
        }
        w.first = lane < kAwRows ? w.prefix_steps + sum - mine : INT32_MAX;
        w.steps = w.prefix_steps + __builtin_amdgcn_readlane(sum, kAwRows - 1);
        return w;
    }
};

// kTiles: whether some part takes 128 rows at a time (LDS for it leaves room for one workgroup per compute unit).
template <typename AC, typename QT, typename CT, int HD, bool kTiles>
__global__ __launch_bounds__(kAwThreads, kTiles ? 2 : 1) void attn_shared_kernel(SharedKernelParams c) {
    constexpr int kTilesBytes = kTiles ? TilesShared<HD, 2>::kBytes : 0, kRowsBytes = (int)sizeof(RowsShared<HD>);
    __shared__ __attribute__((aligned(1024))) unsigned char lds[kTilesBytes > kRowsBytes ? kTilesBytes : kRowsBytes];
    __shared__ int wide;
    // the prefix's tiles first; those of one stretch of keys are a multiple of the number of units apart, on one XCD where that is a multiple of eight
    int at = blockIdx.x;
    const int first = c.part[0].units * c.part[0].blocks * c.part[0].pieces, own = at >= first ? 1 : 0;
    if (own) at -= first;
    const SharedPart &part = c.part[own];
    const int unit = at % part.units, rest = at / part.units, block = rest % part.blocks, piece = rest / part.blocks;
    if constexpr (kTiles) {
        if (part.tiles) {
            attn_tiles<CT, HD, 2>(TilesView(c, own), lds, wide, unit, block, piece);
            return;
        }
    }
    attn_rows<AC, QT, CT, HD>(TextsView(c), *reinterpret_cast<RowsShared<HD> *>(lds), unit, block, piece);
}

// Where row r of a key and value head's is, and how many pieces it has.
struct JoinRow {
    int n_pieces;
    bool padding;
    size_t out;
    __device__ JoinRow(const SharedKernelParams &c, int g, int r, int hd, int step) { // step: positions, of 16 rows at a time
        const AttnSharedParams &a = c.a;
        const int group = a.n_heads / a.n_kv, rows = a.n * group, b = r / rows, own = r - b * rows, i = own / group, start = a.start[b];
        padding = start + i < 0;
        out = ((size_t)(b * a.n + i) * a.n_heads + g * group + (own - i * group)) * hd;
        int steps; // of the rows that were taken together
        if (c.part[1].tiles) {
            const int last = start + (min(rows, (own / kAtRows + 1) * kAtRows) - 1) / group;
            steps = last < 0 ? 0 : last / 128 + 1;
        } else {
            const int r0 = r / kAwRows * kAwRows, r1 = min(a.n_seqs * rows, r0 + kAwRows) - 1;
            steps = c.part[0].pieces > 0 ? 0 : (a.prefix_len + step - 1) / step;
            for (int t = r0 / rows; t <= r1 / rows; t++) {
                const int last = a.start[t] + (min(r1, (t + 1) * rows - 1) - t * rows) / group;
                steps += last < 0 ? 0 : last / step + 1;
            }
        }
        n_pieces = c.part[0].pieces + (steps + c.part[1].piece_steps - 1) / c.part[1].piece_steps;
    }
};

// Row r of key and value head g joins its pieces of the prefix and of its text: a workgroup for a row, where there are few.
template <typename QT, int HD, int kRowsStep>
__global__ __launch_bounds__(kAjWaves *kWave) void attn_shared_join_kernel(SharedKernelParams c) {
    __shared__ float part[kAjWaves * (kWave / (HD / 2))][HD];
    const int g = blockIdx.y, r = blockIdx.x, all = gridDim.x;
    const JoinRow row(c, g, r, HD, kRowsStep);
    QT *out = reinterpret_cast<QT *>(c.a.out) + row.out;
    if (c.part[0].pieces == 0 && !c.part[1].tiles && row.n_pieces <= 1) return; // the row is finished
    if (row.padding) {
        if ((int)threadIdx.x < HD) out[threadIdx.x] = (QT)0.0f;
        return;
    }
    join_pieces<QT, HD, kAjWaves>(part, c.ws + ((size_t)g * all + r) * c.slots * (HD + 2), c.slots, row.n_pieces, out);
}

// ... HD / 4 lanes for a row, where there are many: every lane works out the pieces' weights for itself, eight pieces at a time with a running reference point, and adds up four
// dims.  (39040 rows of two pieces: 21 us with a wavefront for each and its sums through LDS.)
template <typename QT, int HD, int kRowsStep>
__global__ __launch_bounds__(256) void attn_shared_join_rows_kernel(SharedKernelParams c, int all) {
    constexpr int kLanes = HD / 4, kRows = 256 / kLanes, kBatch = 4;
    const int g = blockIdx.y, r = blockIdx.x * kRows + (int)threadIdx.x / kLanes, d = ((int)threadIdx.x % kLanes) * 4;
    if (r >= all) return;
    const JoinRow row(c, g, r, HD, kRowsStep);
    if (c.part[0].pieces == 0 && !c.part[1].tiles && row.n_pieces <= 1) return; // the row is finished
    const float *ws = c.ws + ((size_t)g * all + r) * c.slots * (HD + 2);
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

// How a call is cut.  A workgroup of 16 rows takes `rows_fixed` and, with 128 dims, `rows_step` for every step (32 positions, 16 in f32) of its busiest wavefront; one of 128 rows
// `tiles_fixed` and `tiles_step` for every 128 positions; partial results go to memory and back, and a launch joins them.  The numbers of pieces with the least sum are taken.
// The tiles' workgroups start first, the others fill what is left.
SharedPlan plan_attn_shared(const AttnSharedParams &a, int compute_units) {
    SharedPlan c{};
    const int group = a.n_heads / a.n_kv;
    const int64_t rows = (int64_t)a.n * group, all = rows * a.n_seqs;
    const bool f16 = f16_arithmetic(a), q4 = a.cache == kPlaneQ4;
    const double scale = a.head_dim / 128.0;
    const double rows_fixed = 3.0, rows_step = (q4 ? 1.6 : 1.2) * scale, tiles_fixed = 7.0, tiles_step = (q4 ? 2.6 : 1.9) * scale;
    const int step = f16 ? 32 : 16;
    SharedPart &prefix = c.part[0], &own = c.part[1];
    prefix.tiles = f16 && all > 2 * kAwRows;
    own.tiles = f16 && rows > 2 * kAwRows;
    // steps of the longest, and of all
    int longest = 0, prefix_steps = 0;
    int64_t total = 0;
    if (own.tiles) {
        own.units = a.n_kv * a.n_seqs;
        own.blocks = (int)((rows + kAtRows - 1) / kAtRows);
        for (int b = 0; b < a.n_seqs; b++) {
            const int steps = (std::max(0, a.start[b] + a.n) + 127) / 128;
            longest = std::max(longest, steps);
            total += (int64_t)steps * own.blocks;
        }
    } else {
        own.units = a.n_kv;
        own.blocks = (int)((all + kAwRows - 1) / kAwRows);
        const int first = prefix.tiles ? 0 : (a.prefix_len + step - 1) / step;
        for (int t = 0; t < own.blocks; t++) {
            const int64_t r0 = (int64_t)t * kAwRows, r1 = std::min(all, r0 + kAwRows) - 1;
            int steps = first;
            for (int64_t b = r0 / rows; b <= r1 / rows; b++) steps += (std::max(0, a.start[b] + a.n) + step - 1) / step;
            longest = std::max(longest, steps);
            total += steps;
        }
    }
    if (prefix.tiles) {
        prefix.units = a.n_kv;
        prefix.blocks = (int)((all + kAtRows - 1) / kAtRows);
        prefix_steps = (a.prefix_len + 127) / 128;
    }
    const bool tiles = prefix_steps > 0 || own.tiles;
    const int places = compute_units * (a.head_dim == 128 || tiles ? 1 : 2); // (registers, and LDS of tiles)
    const double mean = longest > 0 ? (double)total / own.blocks / (own.tiles ? a.n_seqs : 1) : 0.0;
    const int most_own = std::min(own.tiles ? 16 : kMaxPieces * 3 / 4, (longest + (own.tiles ? 0 : kAwWaves - 1)) / (own.tiles ? 1 : kAwWaves));
    double least = 0.0;
    int pieces[2] = {0, 0};
    for (int n0 = prefix_steps > 0 ? 1 : 0; n0 <= std::min(kMaxPieces / 2, prefix_steps); n0 += 1 + n0 / 4) {
        for (int n1 = longest > 0 ? 1 : 0; n1 <= std::min(most_own, kMaxPieces - n0); n1 += 1 + n1 / 4) {
            const double part = n1 > 0 ? std::min((double)((longest + n1 - 1) / n1), mean) : 0.0; // steps of an average workgroup
            const double us[2] = {tiles_fixed + (n0 > 0 ? (prefix_steps + n0 - 1) / n0 : 0) * tiles_step,
                                  own.tiles ? tiles_fixed + part * tiles_step : rows_fixed + (double)(((int64_t)part + kAwWaves - 1) / kAwWaves) * rows_step};
            const int64_t count[2] = {(int64_t)prefix.units * prefix.blocks * n0, (int64_t)own.units * own.blocks * n1};
            const bool join = n0 > 0 || own.tiles || n1 > 1;
            const double end = makespan(places, count, us) + (join ? 3.0 + (double)all * a.n_kv * (n0 + n1) * (a.head_dim + 2) * 8 / 4.5e6 : 0.0);
            if ((pieces[0] == 0 && pieces[1] == 0) || end < least) {
                least = end;
                pieces[0] = n0;
                pieces[1] = n1;
            }
            if (longest == 0) break;
        }
        if (prefix_steps == 0) break;
    }
    const int steps[2] = {prefix_steps, longest};
    for (int k = 0; k < 2; k++) {
        SharedPart &p = c.part[k];
        p.piece_steps = pieces[k] > 0 ? (steps[k] + pieces[k] - 1) / pieces[k] : 1;
        p.pieces = steps[k] > 0 ? (steps[k] + p.piece_steps - 1) / p.piece_steps : 0;
        p.first_slot = k ? c.part[0].pieces : 0;
    }
    if (prefix.pieces == 0 && !own.tiles) own.pieces = std::max(1, own.pieces); // (nothing but padding: zeros)
    c.joined = prefix.pieces > 0 || own.tiles || own.pieces > 1;
    c.slots = std::max(1, prefix.pieces + own.pieces);
    c.work_floats = c.joined ? (size_t)all * a.n_kv * c.slots * (a.head_dim + 2) : 0;
    for (const SharedPart &p : c.part) c.workgroups += (int64_t)p.units * p.blocks * p.pieces;
    return c;
}

template <typename AC, typename QT, typename CT, int HD>
static void launch_shared(const SharedKernelParams &c, bool joined, hipStream_t s) {
    int64_t n = 0;
    for (const SharedPart &p : c.part) n += (int64_t)p.units * p.blocks * p.pieces;
    if (n > 0) { // (texts in tiles, and nothing but padding: the join's zeros)
        const dim3 grid((unsigned)n), block(kAwThreads);
        bool tiles = false;
        if constexpr (std::is_same_v<AC, half_t>) {
            tiles = (c.part[0].tiles && c.part[0].pieces > 0) || (c.part[1].tiles && c.part[1].pieces > 0);
            if (tiles) hipLaunchKernelGGL((attn_shared_kernel<AC, QT, CT, HD, true>), grid, block, 0, s, c);
        }
        if (!tiles) hipLaunchKernelGGL((attn_shared_kernel<AC, QT, CT, HD, false>), grid, block, 0, s, c);
    }
    if (!joined) return;
    const unsigned rows = (unsigned)(c.a.n * c.a.n_seqs * (c.a.n_heads / c.a.n_kv)), per = 256 / (HD / 4);
    constexpr int kStep = Step<AC, CT, HD>::kPositions;
    if ((int64_t)rows * c.a.n_kv <= 1024) hipLaunchKernelGGL((attn_shared_join_kernel<QT, HD, kStep>), dim3(rows, (unsigned)c.a.n_kv), dim3(kAjWaves * kWave), 0, s, c);
    else hipLaunchKernelGGL((attn_shared_join_rows_kernel<QT, HD, kStep>), dim3((rows + per - 1) / per, (unsigned)c.a.n_kv), dim3(256), 0, s, c, (int)rows);
}
template <typename AC, typename QT, typename CT>
static hipError_t launch_hd(const SharedKernelParams &c, bool joined, hipStream_t s) {
    switch (c.a.head_dim) {
    case 32: launch_shared<AC, QT, CT, 32>(c, joined, s); break;
    case 64: launch_shared<AC, QT, CT, 64>(c, joined, s); break;
    case 128: launch_shared<AC, QT, CT, 128>(c, joined, s); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_attn_shared(const AttnSharedParams &a, const SharedPlan &plan, float *ws, hipStream_t s) {
    SharedKernelParams c{a, ws, plan.slots, {plan.part[0], plan.part[1]}};
    switch (a.cache * 2 + a.f16) {
    case kPlaneF16 * 2: return launch_hd<float, float, half_t>(c, plan.joined, s);
    case kPlaneF16 * 2 + 1: return launch_hd<half_t, half_t, half_t>(c, plan.joined, s);
    case kPlaneF32 * 2: return launch_hd<float, float, float>(c, plan.joined, s);
    case kPlaneF32 * 2 + 1: return launch_hd<float, half_t, float>(c, plan.joined, s);
    case kPlaneQ4 * 2: return launch_hd<float, float, Quant4>(c, plan.joined, s);
    case kPlaneQ4 * 2 + 1: return launch_hd<half_t, half_t, Quant4>(c, plan.joined, s);
    default: return hipErrorInvalidValue;
    }
}

} // namespace rlh
