// api_answers.hip -- entry points of the C ABI for many answers to one prompt (include/rllama_hip.h): attention behind a shared prefix, log
// probabilities of tokens, and products with weights of 8 bits.
#include "api_planes.h"
#include "answers.h"

#include <climits>
#include <cmath>

using namespace rlh;

// Work memory of calls that need more than their operands.  It grows by doubling, and a smaller one is kept until the context ends: a graph that captured a
// call goes on using the one it was captured with.  While the stream is being captured nothing can be allocated: the call is refused.
static int work_reserve(const char *who, rlh_ctx *ctx, AnswerWork &w, size_t bytes) {
    if (bytes <= w.bytes) return RLH_OK;
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    HIP_TRY(hipStreamIsCapturing(ctx->stream, &status));
    if (status != hipStreamCaptureStatusNone) return fail(RLH_ERR_STATE, "%s: %zu bytes of work memory cannot be allocated while the stream is captured: make a call of this size before", who, bytes);
    if (w.count == AnswerWork::kMost) return fail(RLH_ERR_OOM, "%s: work memory has grown too often", who);
    size_t more = 1 << 20;
    while (more < bytes) more *= 2;
    void *p = nullptr;
    const hipError_t e = device_alloc(ctx, &p, more);
    if (e != hipSuccess) return fail(e == hipErrorOutOfMemory ? RLH_ERR_OOM : RLH_ERR_HIP, "%s: work memory of %zu bytes: %s", who, more, hipGetErrorString(e));
    w.kept[w.count++] = p;
    w.bytes = more;
    return RLH_OK;
}

extern "C" int rlh_attn_shared(rlh_tensor *out, const rlh_tensor *q, const rlh_tensor *prefix_k, const rlh_tensor *prefix_v, int prefix_len, const rlh_tensor *cache_k,
                               const rlh_tensor *cache_v, int n_heads, int n_kv_heads, int max_seq_len, const int32_t *start_pos, int n_seqs) {
    const char *who = "rlh_attn_shared";
    if (!out || !q || !cache_k || !cache_v) return fail(RLH_ERR_INVALID, "%s: NULL argument", who);
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0) return fail(RLH_ERR_INVALID, "%s: %d heads do not share %d key and value heads evenly", who, n_heads, n_kv_heads);
    if (!start_pos || n_seqs < 1 || n_seqs > kLongMaxSeqs) return fail(RLH_ERR_INVALID, "%s: 1 to %d sequences with a position each", who, kLongMaxSeqs);
    constexpr int kFar = INT32_MAX - 256; // (the kernels add up to a tile to a position)
    if (max_seq_len > kFar || prefix_len > kFar) return fail(RLH_ERR_UNSUPPORTED, "%s: planes of %d and %d positions (%d at most)", who, prefix_len, max_seq_len, kFar);
    if (max_seq_len <= 0 || !holds_plane(cache_k) || cache_v->dtype != cache_k->dtype || cache_v->cols != cache_k->cols || (int64_t)n_seqs * n_kv_heads * max_seq_len != cache_k->rows ||
        cache_v->rows != cache_k->rows) {
        return fail(RLH_ERR_INVALID, "%s: cache planes must be two [n_seqs * n_kv_heads * max_seq_len x head_dim] tensors of one dtype", who);
    }
    const int hd = cache_k->cols;
    if (hd != 32 && hd != 64 && hd != 128) return fail(RLH_ERR_UNSUPPORTED, "%s: head_dim %d (32, 64 and 128 are built)", who, hd);
    if (prefix_len < 0 || (prefix_len > 0 && (!prefix_k || !prefix_v)) || !prefix_k != !prefix_v) return fail(RLH_ERR_INVALID, "%s: a prefix of %d positions needs its two planes", who, prefix_len);
    if (prefix_k && (prefix_k->dtype != cache_k->dtype || prefix_v->dtype != cache_k->dtype || prefix_k->cols != hd || prefix_v->cols != hd || prefix_k->rows != prefix_v->rows ||
                     prefix_k->rows % n_kv_heads != 0 || prefix_len > prefix_k->rows / n_kv_heads)) {
        return fail(RLH_ERR_INVALID, "%s: prefix planes must be two [n_kv_heads * rows x head_dim] tensors of the caches' dtype, rows at least %d", who, prefix_len);
    }
    if (q->rows % n_seqs != 0) return fail(RLH_ERR_INVALID, "%s: %d rows are not the same number for each of %d sequences", who, q->rows, n_seqs);
    if (!q->is_float() || out->dtype != q->dtype || !shaped(q, q->rows, (int64_t)n_heads * hd) || !shaped(out, q->rows, (int64_t)n_heads * hd)) {
        return fail(RLH_ERR_INVALID, "%s: q and out must be [rows x n_heads head_dim], both f16 or both f32", who);
    }
    if (out->p == q->p) return fail(RLH_ERR_INVALID, "%s: q and out must not share memory", who);
    const int n = q->rows / n_seqs;
    for (int b = 0; b < n_seqs; b++)
        if ((int64_t)start_pos[b] + n > max_seq_len) return fail(RLH_ERR_STATE, "%s: sequence %d reaches position %lld, the cache has %d", who, b, (long long)start_pos[b] + n - 1, max_seq_len);
    rlh_ctx *ctx = out->ctx;
    CtxLock lock(ctx);
    lend(ctx, {q, cache_k, cache_v});
    if (prefix_k) lend(ctx, {prefix_k, prefix_v});
    AttnSharedParams p{};
    p.q = q->p;
    p.out = out->p;
    p.f16 = q->dtype == RLH_F16;
    p.exact = ctx->tun.attn_exact;
    p.form = ctx->tun.attn_shared_form;
    if (prefix_k) {
        p.prefix_k = plane_of(prefix_k);
        p.prefix_v = plane_of(prefix_v);
        p.prefix_rows = prefix_k->rows / n_kv_heads;
    }
    p.prefix_len = prefix_len;
    p.cache_k = plane_of(cache_k);
    p.cache_v = plane_of(cache_v);
    p.cache = plane_type(cache_k);
    p.n_heads = n_heads;
    p.n_kv = n_kv_heads;
    p.head_dim = hd;
    p.max_seq_len = max_seq_len;
    p.n = n;
    p.n_seqs = n_seqs;
    bool idle = true; // nothing but padding: zeros, and no position is seen
    for (int b = 0; b < n_seqs; b++) {
        p.start[b] = start_pos[b];
        if ((int64_t)start_pos[b] + n > 0) idle = false;
    }
    if (idle) p.prefix_len = 0;
    const SharedPlan plan = plan_attn_shared(p, ctx->prop.multiProcessorCount);
    const int64_t rows = (int64_t)q->rows * (n_heads / n_kv_heads);
    if (plan.workgroups >= 1 << 23 || n_kv_heads > 65535 || rows > INT32_MAX) return fail(RLH_ERR_UNSUPPORTED, "%s: %lld rows on each of %d key and value heads are more than a launch takes", who, (long long)rows, n_kv_heads);
    const int rc = work_reserve(who, ctx, ctx->ops.shared_work, plan.work_floats * sizeof(float));
    if (rc != RLH_OK) return rc;
    HIP_TRY(launch_attn_shared(p, plan, static_cast<float *>(ctx->ops.shared_work.memory()), ctx->stream));
    return RLH_OK;
}

extern "C" int rlh_token_logprobs(rlh_tensor *logprobs, rlh_tensor *entropy, rlh_tensor *top_ids, rlh_tensor *top_logprobs, const rlh_tensor *logits, const rlh_tensor *tokens,
                                  float temperature) {
    const char *who = "rlh_token_logprobs";
    if (!logits || (!logprobs && !entropy && !top_ids)) return fail(RLH_ERR_INVALID, "%s: logits and a result at least are needed", who);
    if (!logits->is_float()) return fail(RLH_ERR_INVALID, "%s: logits must be f16 or f32", who);
    const int rows = logits->rows;
    if (!logprobs != !tokens || (tokens && (tokens->dtype != RLH_I32 || tokens->rows != rows || logprobs->dtype != RLH_F32 || !shaped(logprobs, rows, tokens->cols)))) {
        return fail(RLH_ERR_INVALID, "%s: tokens i32 [rows x m] and logprobs f32 of that shape are needed, or neither", who);
    }
    if (entropy && (entropy->dtype != RLH_F32 || !shaped(entropy, rows, 1))) return fail(RLH_ERR_INVALID, "%s: entropy must be f32 [rows x 1]", who);
    if (!top_ids != !top_logprobs || (top_ids && (top_ids->dtype != RLH_I32 || top_ids->rows != rows || top_logprobs->dtype != RLH_F32 || !shaped(top_logprobs, rows, top_ids->cols)))) {
        return fail(RLH_ERR_INVALID, "%s: top_ids i32 [rows x k] and top_logprobs f32 of that shape are needed, or neither", who);
    }
    if (top_ids && top_ids->cols > logits->cols) return fail(RLH_ERR_INVALID, "%s: %d alternatives of %d entries", who, top_ids->cols, logits->cols);
    if (top_ids && top_ids->cols > kMaxTop) return fail(RLH_ERR_UNSUPPORTED, "%s: %d alternatives (%d at most)", who, top_ids->cols, kMaxTop);
    if (!(temperature >= 1e-30f && temperature <= 1e30f)) return fail(RLH_ERR_INVALID, "%s: temperature %g (1e-30 to 1e30)", who, (double)temperature);
    const rlh_tensor *const all[] = {logprobs, entropy, top_ids, top_logprobs, logits, tokens};
    for (int i = 0; i < 4; i++)
        for (int j = i + 1; j < 6; j++)
            if (all[i] && all[j] && all[i]->p == all[j]->p) return fail(RLH_ERR_INVALID, "%s: results must not share memory with each other or the operands", who);
    rlh_ctx *ctx = (logprobs ? logprobs : entropy ? entropy : top_ids)->ctx;
    CtxLock lock(ctx);
    lend(ctx, {logits});
    for (const rlh_tensor *t : {tokens, (const rlh_tensor *)logprobs, (const rlh_tensor *)entropy, (const rlh_tensor *)top_ids, (const rlh_tensor *)top_logprobs})
        if (t) lend(ctx, {t});
    LogprobsParams p{};
    p.logits = logits->p;
    p.f16 = logits->dtype == RLH_F16;
    p.rows = rows;
    p.vocab = logits->cols;
    p.temperature = temperature;
    if (tokens) {
        p.tokens = (const int32_t *)tokens->p;
        p.n_tokens = tokens->cols;
        p.logprobs = (float *)logprobs->p;
    }
    if (entropy) p.entropy = (float *)entropy->p;
    if (top_ids) {
        p.top_ids = (int32_t *)top_ids->p;
        p.top_logprobs = (float *)top_logprobs->p;
        p.top = top_ids->cols;
    }
    HIP_TRY(launch_token_logprobs(p, ctx->stream));
    return RLH_OK;
}

extern "C" int rlh_matrix_mul_f8(rlh_tensor *dst, const rlh_tensor *src, const rlh_tensor *weights) {
    const char *who = "rlh_matrix_mul_f8";
    if (!dst || !src || !weights) return fail(RLH_ERR_INVALID, "%s: NULL argument", who);
    if (weights->dtype != RLH_F8_TILES) return fail(RLH_ERR_INVALID, "%s: weights must be 8 bits with a scale for each tile", who);
    if (!src->is_float() && src->dtype != RLH_F8) return fail(RLH_ERR_INVALID, "%s: src must be f16, f32 or 8 bits with a scale for each row's blocks", who);
    if (!dst->is_float() || src->cols != weights->cols || !shaped(dst, src->rows, weights->rows)) return fail(RLH_ERR_INVALID, "%s: src [n x k], weights [m x k] and dst [n x m], f16 or f32, are needed", who);
    if (src->cols > (1 << 24)) return fail(RLH_ERR_UNSUPPORTED, "%s: rows of %d (%d at most)", who, src->cols, 1 << 24);
    if (src->rows > (1 << 26) || weights->rows > (1 << 26)) return fail(RLH_ERR_UNSUPPORTED, "%s: %d rows and %d columns (%d at most of each)", who, src->rows, weights->rows, 1 << 26);
    if (dst->p == src->p || dst->p == weights->p) return fail(RLH_ERR_INVALID, "%s: dst must not share memory with the operands", who);
    rlh_ctx *ctx = dst->ctx;
    CtxLock lock(ctx);
    MatmulF8Params p{};
    p.m = src->rows;
    p.n = weights->rows;
    p.k = src->cols;
    p.y = dst->p;
    p.y_f16 = dst->dtype == RLH_F16;
    p.exact = ctx->tun.gemm_f8_exact;
    p.w = eight_of(weights);
    const int cus = ctx->prop.multiProcessorCount;
    // work memory: the sums of pieces of K, and src in 8 bits where the product does not convert it on the way
    const bool on_the_way = src->dtype != RLH_F8 && matmul_f8_converts(p.m, p.k), before = src->dtype != RLH_F8 && !on_the_way;
    const size_t sums = (matmul_f8_work_floats(p, cus) * sizeof(float) + 15) / 16 * 16, codes = src->count();
    const int rc = work_reserve(who, ctx, ctx->ops.f8_work, sums + (before ? codes + (size_t)p.m * f8_blocks(p.k) * sizeof(float) : 0));
    if (rc != RLH_OK) return rc;
    char *work = static_cast<char *>(ctx->ops.f8_work.memory());
    if (src->dtype == RLH_F8) {
        p.x = eight_of(src);
    } else if (before) {
        uint8_t *at = reinterpret_cast<uint8_t *>(work + sums);
        p.x = {at, reinterpret_cast<float *>(at + codes), 1};
    }
    lend(ctx, {src, weights});
    if (before) HIP_TRY(launch_f8_encode(p.x, src->p, src->dtype == RLH_F16, p.m, p.k, ctx->stream));
    HIP_TRY(launch_matmul_f8(p, on_the_way ? src->p : nullptr, src->dtype == RLH_F16, cus, reinterpret_cast<float *>(work), ctx->stream));
    return RLH_OK;
}
