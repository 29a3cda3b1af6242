// attn_tiles.hip -- rlh_attn_window for many rows: the kernel's launch, and how the work is split (attn_tiles_device.h says how it is done).
#include "kernels.h"
#include "attn_tiles_device.h"

#include <algorithm>

namespace rlh {

// kShares: wavefronts per row group.  Late rows see more keys and start first; a unit's workgroups are a multiple of the number of units apart, on one XCD where that is a
// multiple of eight.
template <typename CT, int HD, int kShares>
__global__ __launch_bounds__(64 * kAtGroups *kShares, 2) void attn_tiles_kernel(AttnCutParams pp) {
    __shared__ __attribute__((aligned(1024))) unsigned char lds[TilesShared<HD, kShares>::kBytes];
    __shared__ int wide;
    attn_tiles<CT, HD, kShares>(WindowView(pp), lds, wide, blockIdx.x, (int)gridDim.y - 1 - (int)blockIdx.y, kShares > 1 ? blockIdx.z : 0);
}

// How the work is split: wavefronts per row group, and pieces of each text, of `piece_steps` tiles.
//
// A workgroup with two wavefronts per row group has a compute unit to itself; of those with one there are two on a compute unit.  Two are taken where the
// workgroups would otherwise leave wavefronts idle: fewer of them than compute units, or at most two each while the first rows of a text see little of it
// and their workgroups end early.  (1 / 2 wavefronts, us, 32 heads of 128: 1024 rows from position 0, 256 workgroups, 23.1 / 21.8; 1500, 384, 36.1 / 32.4;
// 2048, 512, 51.4 / 48.3; over 4 bits 27.9 / 25.8, 43.1 / 37.1 and 59.3 / 55.8.  40 heads, 1700 rows, 560: 46.4 / 53.3; 2048, 640: 56.8 / 64.1.  1500 rows
// that all see 1024 positions, 376: 42.3 / 54.2.)
//
// Pieces (with two wavefronts per row group): a compute unit takes 2.3 us per tile of 128 rows and 128 keys of 128 dims; joining costs 4 us and writing and
// reading the partial results, p * 2 (hd + 2) floats per row and head at about 4.5 bytes per ps.  The number of pieces with the least sum is taken.
// What a call takes is about that and 6.5 us.
struct TilesCut {
    int shares, pieces, piece_steps;
    int most; // pieces of a text of any length
    double us;
};
constexpr int kCutKeys = 128;
static TilesCut cut_tiles(const AttnWindowParams &p, int compute_units) {
    const int group = p.n_heads / p.n_kv;
    const int64_t rows = (int64_t)p.n * group, units = (rows + kAtRows - 1) / kAtRows * p.n_seqs * p.n_kv;
    const int64_t apart = std::min<int64_t>(p.n - 1, (kAtRows - 2) / group + 1); // of a workgroup's rows
    int64_t steps = 1;                                                           // no workgroup has more
    bool uneven = false;
    for (int b = 0; b < p.n_seqs; b++) {
        const int64_t last = (int64_t)p.start[b] + p.n - 1;
        if (last < 0) continue;
        int64_t count = (last + kCutKeys) / kCutKeys;
        if (p.window > 0) count = std::min(count, (p.window - 1 + apart + kCutKeys) / kCutKeys) + (p.sinks + kCutKeys - 1) / kCutKeys;
        if (last >= p.max_seq_len) count++; // the ring's end cuts a tile in two
        steps = std::max(steps, count);
        uneven |= (p.window == 0 || p.window > last) && p.start[b] < p.n;
    }
    const double tile_us = 2.3 * p.head_dim / 128, piece_us = (double)p.n * p.n_heads * p.n_seqs * (p.head_dim + 2) * 8 / 4.5e6;
    int64_t n = 1;
    double best = steps * tile_us * std::max(1.0, (double)units / compute_units);
    for (int64_t c = 2; c <= kMaxPieces && c <= steps && c * units <= 2 * compute_units; c++) {
        const double us = (double)((steps + c - 1) / c) * tile_us * std::max(1.0, (double)(c * units) / compute_units) + 4.0 + c * piece_us;
        if (us < best) {
            best = us;
            n = c;
        }
    }
    TilesCut cut;
    cut.us = 6.5 + best;
    cut.most = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxPieces, 2 * compute_units / units));
    cut.piece_steps = (int)((steps + n - 1) / n);
    cut.pieces = (int)((steps + cut.piece_steps - 1) / cut.piece_steps);
    cut.shares = cut.pieces > 1 || units <= (uneven ? 2 : 1) * compute_units ? 2 : 1;
    return cut;
}

int attn_tiles_rows() { return kAtRows; }

double attn_tiles_us(const AttnWindowParams &p, int compute_units) { return cut_tiles(p, compute_units).us; }

size_t attn_tiles_work_floats(const AttnWindowParams &p, int compute_units) {
    const TilesCut cut = cut_tiles(p, compute_units);
    return cut.pieces > 1 ? (size_t)p.n * p.n_heads * p.n_seqs * cut.most * (p.head_dim + 2) : 0;
}

template <typename CT, int HD>
static void launch_tiles(const AttnCutParams &p, int shares, hipStream_t s) {
    const int rows = p.a.n * (p.a.n_heads / p.a.n_kv);
    const unsigned units = (unsigned)(p.a.n_seqs * p.a.n_kv);
    const dim3 grid(units, (unsigned)((rows + kAtRows - 1) / kAtRows), (unsigned)p.pieces);
    if (shares == 1) {
        hipLaunchKernelGGL((attn_tiles_kernel<CT, HD, 1>), grid, dim3(64 * kAtGroups), 0, s, p);
        return;
    }
    hipLaunchKernelGGL((attn_tiles_kernel<CT, HD, 2>), grid, dim3(128 * kAtGroups), 0, s, p);
    if (p.pieces > 1) launch_attn_join<half_t, HD, kAtRows, kCutKeys>(p, s);
}

hipError_t launch_attn_tiles(const AttnWindowParams &a, int compute_units, float *ws, hipStream_t s) {
    const TilesCut cut = cut_tiles(a, compute_units);
    AttnCutParams p;
    p.a = a;
    p.ws = ws;
    p.pieces = cut.pieces;
    p.piece_steps = cut.piece_steps;
    switch (a.head_dim * 2 + (a.cache == kPlaneQ4)) {
    case 64: launch_tiles<half_t, 32>(p, cut.shares, s); break;
    case 65: launch_tiles<Quant4, 32>(p, cut.shares, s); break;
    case 128: launch_tiles<half_t, 64>(p, cut.shares, s); break;
    case 129: launch_tiles<Quant4, 64>(p, cut.shares, s); break;
    case 256: launch_tiles<half_t, 128>(p, cut.shares, s); break;
    case 257: launch_tiles<Quant4, 128>(p, cut.shares, s); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

} // namespace rlh
