// attn_shared.hip -- attention of a batch of texts that share a long prefix.
//
// The row at own position p of text b sees the prefix's positions 0 .. P - 1 and the text's 0 .. p:
//   out = (sum over both of w_t v_t) / (sum of w_t),  w_t = exp(q . k_t / sqrt(hd) - m).
// Sums over parts of the positions, each with a reference point m of its own, join into one: so the prefix is one unit of work for the rows of all texts that
// share a key and value head, read once for all of them instead of once per text, and every text's own positions are another.  One launch takes both, cut into pieces of about
// equal time; each leaves (m, sum, O) of its rows in work memory, and a second launch joins them.
//
// A part whose rows per key and value head are few goes 16 rows at a time from memory into registers (attn_rows_device.h), one with many through tiles of keys in LDS for 128 rows
// (attn_tiles_device.h, f16 arithmetic): the functions of rlh_attn_window, with other positions and other places for results.
#include "kernels.h"
#include "answers.h"
#include "attn_rows_device.h"
#include "attn_tiles_device.h"

#include <algorithm>

namespace rlh {

// One of the two parts: the prefix, or the texts' own positions.
struct SharedPart {
    int blocks;      // of rows, of a unit
    int units;       // the prefix: n_kv; own positions: n_seqs * n_kv
    int pieces, piece_steps;
    int first_slot;  // of its pieces' places in work memory
    int tiles;       // whether 128 rows at a time
};
struct SharedKernelParams {
    AttnSharedParams a;
    float *ws; // for every row of every key and value head the pairs (m, sum) of all its pieces, then the sums O of each
    int slots; // places for pieces
    SharedPart part[2];
};

// A part as the kernels see it.  All rows of the prefix's part are at the prefix's last position.
struct PartParams {
    static constexpr int window = 0, sinks = 0;
    const void *q;
    void *out;
    PlaneRef cache_k, cache_v;
    int n_heads, n_kv, max_seq_len, n;
};
struct SharedView {
    static constexpr bool kPartial = true;
    PartParams p;
    const AttnSharedParams &a;
    int own; // 0: the prefix, 1: the texts' own positions
    float *ws;
    int pieces, piece_steps, first_slot;
    __device__ SharedView(const SharedKernelParams &c, int part)
        : p{c.a.q, c.a.out, part ? c.a.cache_k : c.a.prefix_k, part ? c.a.cache_v : c.a.prefix_v, c.a.n_heads, c.a.n_kv, part ? c.a.max_seq_len : c.a.prefix_rows, part ? c.a.n : c.a.n * c.a.n_seqs},
          a(c.a), own(part), ws(c.ws), pieces(c.slots), piece_steps(c.part[part].piece_steps), first_slot(c.part[part].first_slot) {}
    __device__ int start(int b) const { return own ? a.start[b] : a.prefix_len - 1; }
    __device__ int position(int start, int i) const { return own ? start + i : start; }
    __device__ float *partials(int unit, int rows, int r, int hd) const { // a row's place among those of all texts
        const int b = unit / a.n_kv, g = unit - b * a.n_kv;
        return ws + ((size_t)g * (a.n_seqs * a.n * (a.n_heads / a.n_kv)) + (size_t)b * rows + r) * pieces * (hd + 2);
    }
};

// kTiles: whether some part takes 128 rows at a time (LDS for it leaves room for one workgroup per compute unit).
template <typename AC, typename QT, typename CT, int HD, bool kTiles>
__global__ __launch_bounds__(kAwThreads, kTiles ? 2 : 1) void attn_shared_kernel(SharedKernelParams c) {
    constexpr int kTilesBytes = kTiles ? TilesShared<HD, 2>::kBytes : 0, kRowsBytes = (int)sizeof(RowsShared<HD>);
    __shared__ __attribute__((aligned(1024))) unsigned char lds[kTilesBytes > kRowsBytes ? kTilesBytes : kRowsBytes];
    __shared__ int wide;
    // the prefix's pieces first; those of one stretch of keys are a multiple of the number of units apart, on one XCD where that is a multiple of eight
    int at = blockIdx.x;
    const int first = c.part[0].units * c.part[0].blocks * c.part[0].pieces, own = at >= first ? 1 : 0;
    if (own) at -= first;
    const SharedPart &part = c.part[own];
    const int unit = at % part.units, rest = at / part.units, block = rest % part.blocks, piece = rest / part.blocks;
    const SharedView view(c, own);
    if constexpr (kTiles) {
        if (part.tiles) {
            attn_tiles<CT, HD, 2>(view, lds, wide, unit, block, piece);
            return;
        }
    }
    attn_rows<AC, QT, CT, HD>(view, *reinterpret_cast<RowsShared<HD> *>(lds), unit, block, piece);
}

// Row r of key and value head g joins its pieces of the prefix and of its text.
template <typename QT, int HD, int kRowsStep, int kShare>
__global__ __launch_bounds__(kAjWaves *kWave) void attn_shared_join_kernel(SharedKernelParams c) {
    __shared__ float part[kAjWaves * (kWave / (HD / 2))][HD];
    const AttnSharedParams &a = c.a;
    const int group = a.n_heads / a.n_kv, rows = a.n * group, all = a.n_seqs * rows;
    const int g = blockIdx.y, r = blockIdx.x * (kAjWaves / kShare) + (int)(threadIdx.x / kWave) / kShare;
    if (kShare > 1 ? r >= all : blockIdx.x * kAjWaves >= all) return;
    const int at = min(r, all - 1), b = at / rows, own = at - b * rows, i = own / group, start = a.start[b];
    const int block = c.part[1].tiles ? kAtRows : kAwRows, step = c.part[1].tiles ? 128 : kRowsStep;
    const int last = start + (min(rows, (own / block + 1) * block) - 1) / group; // of the rows that were taken together
    int n_pieces = c.part[0].pieces;
    if (last >= 0) n_pieces += ((last + step) / step + c.part[1].piece_steps - 1) / c.part[1].piece_steps;
    QT *out = reinterpret_cast<QT *>(a.out) + ((size_t)(b * a.n + i) * a.n_heads + g * group + (own - i * group)) * HD;
    const bool idle = r >= all, padding = start + i < 0;
    if (kShare > 1 ? padding : false) { // (all threads have the same row)
        if ((int)threadIdx.x < HD) out[threadIdx.x] = (QT)0.0f;
        return;
    }
    __shared__ QT spare[HD];
    join_pieces<QT, HD, kShare>(part, c.ws + ((size_t)g * all + at) * c.slots * (HD + 2), c.slots, max(1, padding ? 1 : n_pieces), idle || padding ? spare : out);
    if (kShare == 1 && padding && !idle) {
        const int lane = threadIdx.x & (kWave - 1);
        for (int e = lane; e < HD; e += kWave) out[e] = (QT)0.0f;
    }
}

static bool f16_arithmetic(const AttnSharedParams &p) { return p.f16 && p.cache != kPlaneF32; }

// How a call is cut.  Times of one workgroup, with 128 dims: 0.35 us per step of 32 positions of 16 rows (0.5 per 16 positions in f32), 2.3 us per step of 128 positions of 128 rows.
static SharedKernelParams plan_shared(const AttnSharedParams &a, int compute_units) {
    SharedKernelParams c{};
    c.a = a;
    const int group = a.n_heads / a.n_kv;
    const int64_t rows = (int64_t)a.n * group, all = rows * a.n_seqs;
    const bool f16 = f16_arithmetic(a);
    int longest = 0;
    double keys = 0.0; // of all texts
    for (int b = 0; b < a.n_seqs; b++) {
        const int last = std::max(0, a.start[b] + a.n);
        longest = std::max(longest, last);
        keys += last;
    }
    const double scale = a.head_dim / 128.0;
    double step_us[2];
    int steps[2];
    for (int k = 0; k < 2; k++) {
        SharedPart &p = c.part[k];
        const int64_t of_unit = k ? rows : all;
        p.tiles = f16 && of_unit > 2 * kAwRows;
        const int per = p.tiles ? kAtRows : kAwRows, step = p.tiles ? 128 : f16 ? 32 : 16, length = k ? longest : a.prefix_len;
        p.units = k ? a.n_kv * a.n_seqs : a.n_kv;
        p.blocks = (int)((of_unit + per - 1) / per);
        steps[k] = (length + step - 1) / step;
        step_us[k] = (p.tiles ? 2.3 : f16 ? 0.35 : 0.5) * scale;
    }
    const double own_share = longest > 0 ? keys / ((double)longest * a.n_seqs) : 0.0; // of the steps of texts as long as the longest
    const double total = (double)c.part[0].units * c.part[0].blocks * steps[0] * step_us[0] + (double)c.part[1].units * c.part[1].blocks * steps[1] * step_us[1] * own_share;
    const double piece_us = std::max(3.0, total / compute_units);
    for (int k = 0; k < 2; k++) {
        SharedPart &p = c.part[k];
        const int most = k ? std::max(1, kMaxPieces - c.part[0].pieces) : kMaxPieces * 3 / 4;
        const int n = steps[k] > 0 ? std::max(1, std::min({(int)(steps[k] * step_us[k] / piece_us + 0.999), most, steps[k]})) : 0;
        p.piece_steps = n > 0 ? (steps[k] + n - 1) / n : 1;
        p.pieces = steps[k] > 0 ? (steps[k] + p.piece_steps - 1) / p.piece_steps : 0;
        p.first_slot = k ? c.part[0].pieces : 0;
    }
    c.slots = std::max(1, c.part[0].pieces + c.part[1].pieces);
    return c;
}

size_t attn_shared_work_floats(const AttnSharedParams &a, int compute_units) {
    return (size_t)a.n_seqs * a.n * a.n_heads * plan_shared(a, compute_units).slots * (a.head_dim + 2);
}

int64_t attn_shared_workgroups(const AttnSharedParams &a, int compute_units) {
    const SharedKernelParams c = plan_shared(a, compute_units);
    int64_t n = 0;
    for (const SharedPart &p : c.part) n += (int64_t)p.units * p.blocks * p.pieces;
    return n;
}

template <typename AC, typename QT, typename CT, int HD>
static void launch_shared(const SharedKernelParams &c, hipStream_t s) {
    int64_t n = 0;
    for (const SharedPart &p : c.part) n += (int64_t)p.units * p.blocks * p.pieces;
    if (n > 0) {
        const dim3 grid((unsigned)n), block(kAwThreads);
        bool tiles = false;
        if constexpr (std::is_same_v<AC, half_t>) {
            tiles = (c.part[0].tiles && c.part[0].pieces > 0) || (c.part[1].tiles && c.part[1].pieces > 0);
            if (tiles) hipLaunchKernelGGL((attn_shared_kernel<AC, QT, CT, HD, true>), grid, block, 0, s, c);
        }
        if (!tiles) hipLaunchKernelGGL((attn_shared_kernel<AC, QT, CT, HD, false>), grid, block, 0, s, c);
    }
    const unsigned rows = (unsigned)(c.a.n * c.a.n_seqs * (c.a.n_heads / c.a.n_kv));
    constexpr int kStep = Step<AC, CT, HD>::kPositions;
    if ((int64_t)rows * c.a.n_kv <= 1024) hipLaunchKernelGGL((attn_shared_join_kernel<QT, HD, kStep, kAjWaves>), dim3(rows, (unsigned)c.a.n_kv), dim3(kAjWaves * kWave), 0, s, c);
    else hipLaunchKernelGGL((attn_shared_join_kernel<QT, HD, kStep, 1>), dim3((rows + kAjWaves - 1) / kAjWaves, (unsigned)c.a.n_kv), dim3(kAjWaves * kWave), 0, s, c);
}
template <typename AC, typename QT, typename CT>
static hipError_t launch_hd(const SharedKernelParams &c, hipStream_t s) {
    switch (c.a.head_dim) {
    case 32: launch_shared<AC, QT, CT, 32>(c, s); break;
    case 64: launch_shared<AC, QT, CT, 64>(c, s); break;
    case 128: launch_shared<AC, QT, CT, 128>(c, s); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_attn_shared(const AttnSharedParams &a, int compute_units, float *ws, hipStream_t s) {
    SharedKernelParams c = plan_shared(a, compute_units);
    c.ws = ws;
    switch (a.cache * 2 + a.f16) {
    case kPlaneF16 * 2: return launch_hd<float, float, half_t>(c, s);
    case kPlaneF16 * 2 + 1: return launch_hd<half_t, half_t, half_t>(c, s);
    case kPlaneF32 * 2: return launch_hd<float, float, float>(c, s);
    case kPlaneF32 * 2 + 1: return launch_hd<float, half_t, float>(c, s);
    case kPlaneQ4 * 2: return launch_hd<float, float, Quant4>(c, s);
    case kPlaneQ4 * 2 + 1: return launch_hd<half_t, half_t, Quant4>(c, s);
    default: return hipErrorInvalidValue;
    }
}

} // namespace rlh
