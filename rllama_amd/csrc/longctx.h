// longctx.h -- launch interface of the kernels for long contexts and drafted tokens (internal to librllama_hip.so).
#pragma once

#include "q4.h"

namespace rlh {

constexpr int kLongMaxSeqs = 256; // positions travel as kernel arguments: 1 KiB of the 4 KiB a launch may carry
constexpr int64_t kLongMaxPosition = INT32_MAX - 255; // the kernels add up to a tile of positions to one in 32 bits

enum PlaneType { kPlaneF16 = 0, kPlaneF32 = 1, kPlaneQ4 = 2 };

struct QkvAppendParams {
    PlaneRef qkv, q;       // rows of a projection, rows of queries (f16 or f32)
    int f16;               // type of both
    const float *q_norm, *k_norm; // [head_dim] or null
    float eps;
    const float *freqs;    // [positions x head_dim]: pairs (cos, sin)
    int halves;            // a pair is columns (j, j + head_dim / 2) instead of (2 j, 2 j + 1)
    PlaneRef cache_k, cache_v;
    int cache;             // PlaneType
    int n_heads, n_kv, head_dim, max_seq_len, sinks;
    int n, n_seqs;
    int32_t start[kLongMaxSeqs];
};
hipError_t launch_qkv_append(const QkvAppendParams &p, hipStream_t s);

struct AttnWindowParams {
    const void *q;
    void *out;
    int f16;               // type of q and out
    PlaneRef cache_k, cache_v;
    int cache;             // PlaneType
    int n_heads, n_kv, head_dim, max_seq_len;
    int n, n_seqs;
    int window, sinks;     // window 0: everything up to the row's own position
    int exact;             // only the form that rounds nothing but the result
    int32_t start[kLongMaxSeqs];
};
// rows of one key and value head (n * n_heads / n_kv) that a launch takes; 0: too many sequences and heads
int64_t attn_window_most_rows(const AttnWindowParams &p, int compute_units);
// work memory for partial results where this call cuts its texts: enough for as many pieces as texts of any length are cut into, at most 512 workgroups' rows (34 MB)
size_t attn_window_work_floats(const AttnWindowParams &p, int compute_units);
// the form for many rows (attn_tiles.hip): which calls it takes, its work memory and its launch
int attn_tiles_rows(); // of a workgroup
double attn_tiles_us(const AttnWindowParams &p, int compute_units); // about what a call takes
size_t attn_tiles_work_floats(const AttnWindowParams &p, int compute_units);
hipError_t launch_attn_tiles(const AttnWindowParams &p, int compute_units, float *ws, hipStream_t s);
hipError_t launch_attn_window(const AttnWindowParams &p, int compute_units, float *ws, hipStream_t s);

// elements between f16, f32 and 4 bits; count a multiple of 32 where one side has 4 bits
hipError_t launch_plane_convert(const PlaneRef &dst, int dst_type, const PlaneRef &src, int src_type, size_t count, hipStream_t s);

hipError_t launch_softmax_rows(float *probs, const void *logits, int logits_f16, int rows, int vocab, float temperature, hipStream_t s);

struct VerifyParams {
    const float *target, *draft; // [n_seqs * (k + 1) x vocab], [n_seqs * k x vocab] or null
    const int32_t *drafted;      // [n_seqs x k]
    const float *uniforms;       // [n_seqs x (k + 1)]
    int32_t *out;                // [n_seqs x (k + 2)]
    int n_seqs, k, vocab;
};
hipError_t launch_verify_draft(const VerifyParams &p, hipStream_t s);

} // namespace rlh
