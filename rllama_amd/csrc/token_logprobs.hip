// token_logprobs.hip -- log probabilities of given tokens, the entropy of rows of logits and their most probable tokens.
//
// With z = (x - m) / T, m the row's largest, and s the sum of exp(z) over all entries but one that is the largest:
//   log p(t) = z_t - log(1 + s),   entropy = log(1 + s) - (sum of z exp(z)) / (1 + s).
// Leaving one largest entry out of the sum keeps what is small beside it: where a token is all but certain, its log probability and the entropy are as exact as
// the others' weights are (a sum that holds the 1 loses everything below 2^-24 of it).
//
// One workgroup per row, of 256 to 1024 threads.  A row of up to 32768 entries is read once and stays in registers, up to 128 bytes per thread; a longer one is read
// three times, the second and third time from the caches.
//
// Measured: 16 rows of 32000 in f32 with five alternatives 7.8 us, the latency of a row on one compute unit; 2048 rows in f16 with twenty 41 us, 3.2 TB/s: the vector ALU is busy for 61 %
// (an exponential, two sums and a maximum for each entry).
//
// The k most probable: the 64 groups of threads have a largest entry each, and the k-th largest of those bounds the k-th largest entry from below, since k groups hold an
// entry that large.  What reaches the bound (about k ln(64 / (64 - k)) / (k / 64) of 32000 random entries) goes to a list in LDS, and an entry's place is the number
// of those in front of it.  Lists that overflow: of rows with many entries equal to the bound (masks) those above it, and then the first equal ones in order of their ids.
// Where those above it are too many as well (they lie side by side, in fewer than k groups), the k-th largest of the threads' own entries is a closer bound, and
// where that is not enough, one entry after the other.
#include "kernels.h"
#include "answers.h"

#include <algorithm>
#include <type_traits>

namespace rlh {

constexpr int kTlList = 256;
constexpr int kTlGroups = 64;
constexpr int kTlCrowd = 700; // rows from which on small workgroups gain

template <int kCtrl, int kRowMask = 0xf>
__device__ __forceinline__ float dpp_max(float v) { // (lanes whose row is masked out keep v)
    const int x = __builtin_bit_cast(int, v);
    return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(x, x, kCtrl, kRowMask, 0xf, false)));
}
__device__ __forceinline__ float wave_top(float v) { // the wavefront's largest, in all lanes
    v = dpp_max<kDppRowMirror>(dpp_max<kDppRowHalfMirror>(dpp_max<kDppQuadPerm2301>(dpp_max<kDppQuadPerm1032>(v))));
    v = dpp_max<kDppRowBcast31, 0xc>(dpp_max<kDppRowBcast15, 0xa>(v));
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// kN entries of a row, sixteen bytes at most.  Rows of any length: only the element's own alignment.
template <typename T, int kN>
struct RowPiece {
    typedef T any __attribute__((ext_vector_type(kN), aligned(sizeof(T))));
    typedef T vec __attribute__((ext_vector_type(kN)));
    vec v;
    __device__ __forceinline__ void load(const T *x, int64_t i, int n) { // -infinity behind the row's end
        if (i <= (int64_t)n - kN) {
            v = *reinterpret_cast<const any *>(x + i);
        } else {
#pragma unroll
            for (int j = 0; j < kN; j++) v[j] = i + j < n ? x[i + j] : (T)-INFINITY;
        }
    }
    __device__ __forceinline__ float at(int j) const { return (float)v[j]; }
    // Keeps the bytes as they are from one pass over the pieces to the next (converted once for all passes they took four times the registers, and half of the
    // workgroups fit a compute unit).
    __device__ __forceinline__ void hold() {
        typedef std::conditional_t<sizeof(v) == 4, uint32_t, std::conditional_t<sizeof(v) == 8, unsigned long long, uint4_t>> words;
        words w = __builtin_bit_cast(words, v);
        asm volatile("" : "+v"(w));
        v = __builtin_bit_cast(vec, w);
    }
};

// larger values first, of equal ones the lower id; all keys differ
__device__ __forceinline__ unsigned long long logit_key(float v, int id) {
    const uint32_t w = __builtin_bit_cast(uint32_t, v + 0.0f); // (zeros of either kind are equal)
    return ((unsigned long long)(w & 0x80000000u ? ~w : w | 0x80000000u) << 32) | (uint32_t)~(uint32_t)id;
}
__device__ __forceinline__ float key_logit(unsigned long long key) {
    const uint32_t w = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, w & 0x80000000u ? w & 0x7fffffffu : ~w);
}

// kKeep: pieces of kN entries that a thread keeps; 0: rows of any length.  kMany: of more rows than compute units, two to a compute unit.  c2 = log2(e) / T, inverse = 1 / T.
template <typename T, int kThreads, int kN, int kKeep, bool kMany>
__global__ __launch_bounds__(kThreads, kMany && kN > 2 ? 8 : 4) void token_logprobs_kernel(LogprobsParams p, float c2, float inverse) {
    typedef RowPiece<T, kN> Piece;
    constexpr int kStep = kThreads * kN, kWaves = kThreads / kWave, kLanes = kThreads / kTlGroups;
    __shared__ __attribute__((aligned(16))) float group_top[kTlGroups];
    __shared__ float group_low[kTlGroups], sums[3][kWaves];
    __shared__ unsigned long long list[kTlList], sh_best;
    __shared__ int sh_count, sh_holders, holders[kThreads], sh_ties[kWaves];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int row = blockIdx.x, vocab = p.vocab;
    const T *x = reinterpret_cast<const T *>(p.logits) + (size_t)row * vocab;
    Piece kept[kKeep > 0 ? kKeep : 1];
    // f(piece, id of its first entry) over the thread's pieces
    auto pieces = [&](auto f) __attribute__((always_inline)) {
        if constexpr (kKeep > 0) {
#pragma unroll
            for (int k = 0; k < kKeep; k++) {
                if (k * kStep >= vocab) break; // (behind the row: one row of 10000 7.6 -> 6.4 us)
                if (kMany) kept[k].hold();
                f(kept[k], k * kStep + tid * kN);
                if (kMany) __builtin_amdgcn_sched_barrier(0); // (one after the other, or each piece takes registers of its own for what is worked out)
            }
        } else {
            for (int64_t i = (int64_t)tid * kN; i < vocab; i += kStep) {
                Piece piece;
                piece.load(x, i, vocab);
                f(piece, i);
            }
        }
    };
    // the same, from memory again
    auto reread = [&](auto f) __attribute__((always_inline)) {
#pragma unroll 1
        for (int64_t i = (int64_t)tid * kN; i < vocab; i += kStep) {
            Piece piece;
            piece.load(x, i, vocab);
            f(piece, i);
        }
    };
    if constexpr (kKeep > 0) {
#pragma unroll
        for (int k = 0; k < kKeep; k++) kept[k].load(x, k * kStep + tid * kN, vocab);
    }
    // the first of the tokens asked for, on their way beside the row
    const int token = tid < p.n_tokens ? p.tokens[(size_t)row * p.n_tokens + tid] : -1;
    const float token_logit = token >= 0 && token < vocab ? (float)x[token] : 0.0f;
    // ---- the largest entry, of the thread, of its group and of the row
    float mine = -INFINITY;
    pieces([&](const Piece &piece, auto) {
        typename Piece::vec t = piece.v;
#pragma unroll
        for (int n = kN / 2; n > 0; n /= 2)
#pragma unroll
            for (int j = 0; j < n; j++) t[j] = __builtin_elementwise_max(t[j], t[j + n]);
        mine = fmaxf(mine, (float)t[0]);
    });
    {
        float top = dpp_max<kDppQuadPerm2301>(dpp_max<kDppQuadPerm1032>(mine));
        if constexpr (kLanes >= 8) top = dpp_max<kDppRowHalfMirror>(top);
        if constexpr (kLanes >= 16) top = dpp_max<kDppRowMirror>(top);
        static_assert(kLanes == 16 || kLanes == 8 || kLanes == 4, "1024, 512 or 256 threads");
        if (tid % kLanes == 0) group_top[tid / kLanes] = top;
    }
    if (tid < kTlList) list[tid] = 0;
    if (tid == 0) sh_count = sh_holders = 0;
    __syncthreads();
    const float m = wave_top(group_top[lane]), base = m > -INFINITY ? m : 0.0f;
    if (p.top > 0) { // the groups whose entry is among the k largest: a group's threads compare its own with a few others each
        const float own = group_top[tid / kLanes];
        float above = 0.0f;
#pragma unroll
        for (int g = 0; g < kTlGroups / kLanes; g += 4) {
            const float4_t other = *reinterpret_cast<const float4_t *>(&group_top[tid % kLanes * (kTlGroups / kLanes) + g]);
#pragma unroll
            for (int j = 0; j < 4; j++) above += other[j] > own ? 1.0f : 0.0f;
        }
        above = group_sum<kLanes>(above);
        if (tid % kLanes == 0) group_low[tid / kLanes] = above < (float)p.top ? -own : -INFINITY;
    }
    // ---- the sums.  f16: z = x c2 - m c2 in one operation; m c2 was rounded, which shifts all z by the same `shift`, half a unit of m c2.  f32: the difference first, since
    // m c2 may not be representable, and half of it, since the difference of two numbers may not be either.  (A bound keeps 0 * infinity out of the second sum.)
    // f16 with |m c2| from 2^24 on (a low temperature), where that unit grows without bound: numbers of 11 bits that differ from m differ by 2^-11 of it at least, so their z
    // are below -2^12 and their weights 0 whatever c2 is.  A power of two in its place, m c2 between 2^23 and 2^24, gives the same sums with no shift.
    const bool far = sizeof(T) == 2 && fabsf(base) * c2 >= 16777216.0f;
    const float by = far ? ldexpf(1.0f, 24 - __builtin_amdgcn_frexp_expf(base)) : c2;
    const float mc = sizeof(T) == 2 ? base * by : 0.0f, shift = sizeof(T) == 2 ? fmaf(base, by, -mc) : 0.0f;
    const float half_base = 0.5f * base, c2_twice = 2.0f * c2, inverse_twice = 2.0f * inverse;
    auto exponent = [&](float v) { return sizeof(T) == 2 ? fmaf(v, by, -mc) : fmaf(v, 0.5f, -half_base) * c2_twice; };
    float s = 0.0f, u = 0.0f, count = 0.0f;
    if (mine < m || !(m > -INFINITY)) {
        pieces([&](const Piece &piece, auto) {
#pragma unroll
            for (int j = 0; j < kN; j++) {
                const float z = exponent(piece.at(j)), e = __builtin_amdgcn_exp2f(z);
                s += e;
                u = fmaf(e, fmaxf(z, -300.0f), u);
            }
        });
    } else { // the thread holds a largest entry: one is left out
        count = 1.0f;
        pieces([&](const Piece &piece, auto) {
#pragma unroll
            for (int j = 0; j < kN; j++) {
                const bool out = count > 0.0f && piece.at(j) == m;
                const float z = exponent(piece.at(j)), e = out ? 0.0f : __builtin_amdgcn_exp2f(z);
                if (out) count = 0.0f;
                s += e;
                u = fmaf(e, fmaxf(z, -300.0f), u);
            }
        });
        count = 1.0f;
    }
    s = wave_sum(s);
    u = wave_sum(u);
    count = wave_sum(count);
    if (lane == 0) {
        sums[0][wave] = s;
        sums[1][wave] = u;
        sums[2][wave] = count;
    }
    __syncthreads();
    s = u = count = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        s += sums[0][w];
        u += sums[1][w];
        count += sums[2][w];
    }
    const bool none = !(m > -INFINITY), odd = !(s < INFINITY) || m == INFINITY; // (a NaN is in the sum)
    constexpr float kLn2 = 0.69314718055994530942f;
    const float e_top = __builtin_amdgcn_exp2f(shift);
    const float others = fmaf(fmaxf(count - 1.0f, 0.0f), e_top, s) / e_top; // (a thread each left out one of several that are the largest)
    const float log_s = log1pf(others), u_top = (u - shift * s) / e_top;
    auto logprob = [&](float v) { return odd ? NAN : none ? -INFINITY : fmaf(fmaf(v, 0.5f, -half_base), inverse_twice, -log_s); };
    if (tid == 0 && p.entropy) p.entropy[row] = odd ? NAN : none ? 0.0f : log_s - kLn2 * u_top / (1.0f + others);
    for (int i = tid; i < p.n_tokens; i += kThreads) {
        const int id = i == tid ? token : p.tokens[(size_t)row * p.n_tokens + i];
        p.logprobs[(size_t)row * p.n_tokens + i] = id < 0 ? 0.0f : id < vocab ? logprob(i == tid ? token_logit : (float)x[id]) : odd ? NAN : -INFINITY;
    }
    if (p.top == 0) return;
    int32_t *ids = p.top_ids + (size_t)row * p.top;
    float *logprobs = p.top_logprobs + (size_t)row * p.top;
    if (odd) {
        if (tid < p.top) {
            ids[tid] = -1;
            logprobs[tid] = NAN;
        }
        return;
    }
    // ---- the most probable
    float bound = -wave_top(group_low[lane]); // the least of theirs
    // Threads that hold such an entry note themselves; their entries are then shared out, one to a thread, and read again.  (Each looking through its own
    // took 4 us: nearly every wavefront has one of them.)
    if (mine >= bound) holders[atomicAdd(&sh_holders, 1)] = tid;
    __syncthreads();
    typedef std::conditional_t<(kKeep > 0), int, int64_t> index_t;
    const index_t each = kKeep > 0 ? kKeep * kN : (int)(((int64_t)vocab + kStep - 1) / kStep) * kN;
    auto collect = [&](bool equal_ones) __attribute__((always_inline)) {
        const index_t all = (index_t)sh_holders * each;
        for (index_t e = tid; e < all; e += kThreads) {
            const int h = (int)(e / each), j = (int)(e - (index_t)h * each);
            const index_t id = (index_t)(j / kN) * kStep + holders[h] * kN + j % kN;
            if (id >= vocab) continue;
            const float v = (float)x[id];
            if (equal_ones ? v >= bound : v > bound) {
                const int at = atomicAdd(&sh_count, 1);
                if (at < kTlList) list[at] = logit_key(v, (int)id);
            }
        }
    };
    auto count_of = [&](bool equal_ones) __attribute__((always_inline)) {
        collect(equal_ones);
        __syncthreads();
        return sh_count;
    };
    auto again = [&] { // the list is empty
        __syncthreads();
        if (tid == 0) sh_count = 0;
        if (tid < kTlList) list[tid] = 0;
        __syncthreads();
    };
    int found = count_of(true), wanted = p.top; // of the list
    if (found > kTlList) {
        again();
        found = count_of(false);
        bool equal_ones = true; // are left to be added
        if (found > kTlList) {
            again();
            // the k-th largest of the threads' own (32 of 1000 entries side by side, all others masked, in 32000: 300 us one after the other, 33 so)
            if (tid == 0) sh_holders = 0;
            __syncthreads();
            if (mine > bound) holders[atomicAdd(&sh_holders, 1)] = __builtin_bit_cast(int, mine);
            __syncthreads();
            int n = sh_holders, above = 0;
            for (int i = 0; i < n; i++) above += __builtin_bit_cast(float, holders[i]) > mine;
            const float low = wave_top(mine > bound && above < p.top ? -mine : -INFINITY);
            if (lane == 0) sums[0][wave] = low;
            __syncthreads();
            float least = sums[0][0];
#pragma unroll
            for (int w = 1; w < kWaves; w++) least = fmaxf(least, sums[0][w]);
            if (n >= p.top) {
                bound = -least;
                if (tid == 0) sh_holders = 0;
                __syncthreads();
                if (mine >= bound) holders[atomicAdd(&sh_holders, 1)] = tid;
                __syncthreads();
                found = count_of(true);
                equal_ones = false;
                if (found > kTlList) {
                    again();
                    found = count_of(false);
                    equal_ones = true;
                }
            }
        }
        if (found > kTlList) { // one after the other
            unsigned long long below = ~0ull;
            for (int k = 0; k < p.top; k++) {
                if (tid == 0) sh_best = 0;
                __syncthreads();
                unsigned long long best = 0;
                reread([&](const Piece &piece, int64_t i) {
#pragma unroll
                    for (int j = 0; j < kN; j++) {
                        const unsigned long long key = logit_key(piece.at(j), (int)(i + j));
                        if (key < below && key > best && i + j < vocab) best = key;
                    }
                });
                if (best) atomicMax(&sh_best, best);
                __syncthreads();
                below = sh_best;
                __syncthreads();
                if (tid == 0) {
                    ids[k] = (int)~(uint32_t)below;
                    logprobs[k] = logprob(key_logit(below));
                }
            }
            return;
        }
        if (equal_ones) wanted = min(p.top, found);
        // the first ids of entries that equal the bound, a stretch of the row at a time
        const float at_bound = logprob(bound);
        int place = equal_ones ? found : p.top;
        for (int64_t from = 0; place < p.top && from < vocab; from += kStep) {
            Piece piece;
            piece.load(x, from + (int64_t)tid * kN, vocab);
            int n = 0;
#pragma unroll
            for (int j = 0; j < kN; j++) n += piece.at(j) == bound && from + tid * kN + j < vocab;
            int before = n; // of the wavefront's lanes up to this one
#pragma unroll
            for (int off = 1; off < kWave; off <<= 1) {
                const int up = __shfl_up(before, off, kWave);
                if (lane >= off) before += up;
            }
            if (lane == kWave - 1) sh_ties[wave] = before;
            __syncthreads();
            int at = place + before - n;
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                if (w < wave) at += sh_ties[w];
                place += sh_ties[w];
            }
            if (n > 0) {
#pragma unroll
                for (int j = 0; j < kN; j++)
                    if (piece.at(j) == bound && from + tid * kN + j < vocab && at < p.top) {
                        ids[at] = (int)(from + tid * kN + j);
                        logprobs[at++] = at_bound;
                    }
            }
            __syncthreads();
        }
    }
    for (int i = tid; i < found; i += kThreads) {
        const unsigned long long key = list[i];
        int at = 0;
#pragma unroll 1 // (32 places at a time took twice the registers of all that came before, and spilled)
        for (int j = 0; j < found; j += 8) // (places behind the last one are 0)
#pragma unroll
            for (int u = 0; u < 8; u++) at += list[j + u] > key;
        if (at < wanted) {
            ids[at] = (int)~(uint32_t)key;
            logprobs[at] = logprob(key_logit(key));
        }
    }
}

template <typename T, bool kMany>
static void launch_t(const LogprobsParams &p, hipStream_t s) {
    constexpr int kN = 16 / (int)sizeof(T);
    const float c2 = (float)(1.44269504088896340736 / (double)p.temperature), inverse = (float)(1.0 / (double)p.temperature);
    const dim3 grid((unsigned)p.rows);
    // Narrow pieces in short rows, so that 33 groups at least hold entries: 20 or 32 alternatives of 500 entries, or of 2100 in f16, took 85 to 150 us in pieces of sixteen
    // bytes, whose few groups give no bound, and take less than 20 so, as those of other lengths do.
    // A row's time is mostly that of its steps one after the other, whatever its length: many rows go to workgroups as small as their registers allow, up to eight of which
    // share a compute unit (f16, five alternatives: 2048 rows of 32000 41 -> 37 us, of 10000 38.5 -> 21, of 6000 24 -> 15; 800 rows 22.1 / 22.3, 20.9 / 12.7, 13 / 8.6;
    // 400 rows of 32000 13.6 -> 14.1).
    const bool crowd = p.rows > kTlCrowd;
    if (p.vocab <= 2048) hipLaunchKernelGGL((token_logprobs_kernel<T, 256, 2, 4, kMany>), grid, dim3(256), 0, s, p, c2, inverse);
    else if (crowd && p.vocab <= 8192) hipLaunchKernelGGL((token_logprobs_kernel<T, 256, kN, 32 / kN, true>), grid, dim3(256), 0, s, p, c2, inverse);
    else if (crowd && p.vocab <= 16384) hipLaunchKernelGGL((token_logprobs_kernel<T, kN == 8 ? 256 : 512, kN, 8, true>), grid, dim3(kN == 8 ? 256 : 512), 0, s, p, c2, inverse);
    else if (crowd && p.vocab <= 32768 && kN == 8) hipLaunchKernelGGL((token_logprobs_kernel<T, 512, kN, 8, true>), grid, dim3(512), 0, s, p, c2, inverse);
    else if (p.vocab <= 8192) hipLaunchKernelGGL((token_logprobs_kernel<T, 1024, 4, 2, kMany>), grid, dim3(1024), 0, s, p, c2, inverse);
    else if (p.vocab <= 32768) hipLaunchKernelGGL((token_logprobs_kernel<T, 1024, kN, 32 / kN, kMany>), grid, dim3(1024), 0, s, p, c2, inverse);
    else hipLaunchKernelGGL((token_logprobs_kernel<T, 1024, kN, 0, kMany>), grid, dim3(1024), 0, s, p, c2, inverse);
}

hipError_t launch_token_logprobs(const LogprobsParams &all, hipStream_t s) {
    constexpr int kRows = 1 << 21; // of a launch, which takes less than 2^32 threads
    for (int64_t r0 = 0; r0 < all.rows; r0 += kRows) {
        LogprobsParams p = all;
        p.rows = (int)std::min<int64_t>(kRows, all.rows - r0);
        p.logits = static_cast<const char *>(all.logits) + (size_t)r0 * all.vocab * (all.f16 ? 2 : 4);
        if (all.tokens) {
            p.tokens = all.tokens + (size_t)r0 * all.n_tokens;
            p.logprobs = all.logprobs + (size_t)r0 * all.n_tokens;
        }
        if (all.entropy) p.entropy = all.entropy + r0;
        if (all.top > 0) {
            p.top_ids = all.top_ids + (size_t)r0 * all.top;
            p.top_logprobs = all.top_logprobs + (size_t)r0 * all.top;
        }
        if (p.f16) p.rows > 256 ? launch_t<half_t, true>(p, s) : launch_t<half_t, false>(p, s);
        else p.rows > 256 ? launch_t<float, true>(p, s) : launch_t<float, false>(p, s);
    }
    return hipGetLastError();
}

} // namespace rlh
