// answers.h -- launch interface of the kernels for many answers to one prompt (internal to librllama_hip.so): attention behind a shared
// prefix, log probabilities of tokens, tensors and products of 8 bits.
#pragma once

#include "f8.h"
#include "longctx.h"

namespace rlh {

struct AttnSharedParams {
    const void *q;
    void *out;
    int f16;                    // type of q and out
    int exact;                  // nothing is rounded but the result
    int form;                   // 0: what takes less time, 1: 16 rows at a time, 2: tiles
    PlaneRef prefix_k, prefix_v; // [n_kv * prefix_rows x head_dim], of which prefix_len rows of each head are seen by every row
    PlaneRef cache_k, cache_v;  // [n_seqs * n_kv * max_seq_len x head_dim]
    int cache;                  // PlaneType of all four
    int n_heads, n_kv, head_dim, max_seq_len;
    int prefix_len, prefix_rows;
    int n, n_seqs;
    int32_t start[kLongMaxSeqs];
};
// How a call is cut: what goes through tiles, and what 16 rows at a time.  One of them has the prefix, one the texts' own positions.
struct SharedPart {
    int prefix, texts;
    int blocks; // of rows, of a key and value head
    int whole;  // of them the first ones, which are not cut
    int pieces, piece_steps; // of the others
    int first_slot; // of its pieces' places in work memory
};
struct SharedPlan {
    SharedPart part[2];
    int slots;   // places for pieces
    int cut;     // the first row of a head that is cut
    bool joined; // by a second launch
    size_t work_floats;
    int64_t workgroups;
};
SharedPlan plan_attn_shared(const AttnSharedParams &p, int compute_units);
hipError_t launch_attn_shared(const AttnSharedParams &p, const SharedPlan &plan, float *ws, hipStream_t s);

constexpr int kMaxTop = 32; // alternatives of a row
struct LogprobsParams {
    const void *logits;
    int f16;
    int rows, vocab;
    float temperature;
    const int32_t *tokens; // [rows x n_tokens] or null
    int n_tokens;
    float *logprobs;       // [rows x n_tokens] or null
    float *entropy;        // [rows] or null
    int32_t *top_ids;      // [rows x top] or null
    float *top_logprobs;
    int top;
};
hipError_t launch_token_logprobs(const LogprobsParams &p, hipStream_t s);

// f16 or f32 to 8 bits and back
hipError_t launch_f8_encode(const EightRef &dst, const void *src, int src_f16, int rows, int cols, hipStream_t s);
hipError_t launch_f8_decode(void *dst, int dst_f16, const EightRef &src, int rows, int cols, hipStream_t s);

struct MatmulF8Params {
    EightRef x, w; // [m x k] a scale for every row and block, [n x k] a scale for every tile
    void *y;       // [m x n]
    int y_f16;
    int exact; // f16 results of many rows are summed up in f32 as well
    int m, n, k;
};
bool matmul_f8_converts(int m, int k);                                   // whether a product of m rows converts f16 and f32 rows on the way
size_t matmul_f8_work_floats(const MatmulF8Params &p, int compute_units); // sums of pieces of K
// src: f16 or f32 rows that are converted on the way (p.x is not used then), or null
hipError_t launch_matmul_f8(const MatmulF8Params &p, const void *src, int src_f16, int compute_units, float *ws, hipStream_t s);

} // namespace rlh
