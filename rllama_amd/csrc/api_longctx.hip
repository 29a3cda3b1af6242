// api_longctx.hip -- entry points of the C ABI for long contexts and drafted tokens (include/rllama_hip.h): tensors over the caller's
// memory, conversion to and from 4 bits, the append of a projection's rows to the caches, attention with a window, the
// probabilities of rows of logits and the verification of drafted tokens.
#include "api_planes.h"
#include "answers.h"

#include <climits>
#include <cmath>
#include <new>

using namespace rlh;

extern "C" int rlh_tensor_wrap(rlh_ctx *ctx, void *device_memory, int rows, int cols, int dtype, rlh_tensor **out) {
    if (!ctx || !out || !device_memory || rows <= 0 || cols <= 0 || !known_dtype(dtype)) return fail(RLH_ERR_INVALID, "rlh_tensor_wrap: bad argument");
    if (dtype == RLH_Q4 && cols % kQ4Group != 0) return fail(RLH_ERR_INVALID, "rlh_tensor_wrap: %d columns of 4 bits: a multiple of %d is needed", cols, kQ4Group);
    if (dtype >= RLH_F8 && cols % 16 != 0) return fail(RLH_ERR_INVALID, "rlh_tensor_wrap: %d columns of 8 bits: a multiple of 16 is needed", cols);
    if (reinterpret_cast<uintptr_t>(device_memory) % 16 != 0) return fail(RLH_ERR_INVALID, "rlh_tensor_wrap: the memory must be 16-byte aligned");
    *out = nullptr;
    rlh_tensor *t = new (std::nothrow) rlh_tensor();
    if (!t) return fail(RLH_ERR_OOM, "rlh_tensor_wrap: out of host memory");
    t->ctx = ctx;
    t->p = device_memory;
    t->rows = rows;
    t->cols = cols;
    t->dtype = dtype;
    t->capacity = t->bytes();
    t->wrapped = true;
    *out = t;
    return RLH_OK;
}

// `later` waits for what is queued on `earlier`
static int order_streams(const char *who, rlh_ctx *ctx, hipStream_t earlier, hipStream_t later) {
    CtxLock lock(ctx);
    hipEvent_t ev = nullptr;
    hipError_t e = hipEventCreateWithFlags(&ev, hipEventDisableTiming);
    if (e == hipSuccess) e = hipEventRecord(ev, earlier);
    if (e == hipSuccess) e = hipStreamWaitEvent(later, ev, 0);
    if (ev) (void)hipEventDestroy(ev); // (kept by the runtime until it has been passed)
    if (e != hipSuccess) return fail(RLH_ERR_HIP, "%s: %s", who, hipGetErrorString(e));
    return RLH_OK;
}

extern "C" int rlh_wait_stream(rlh_ctx *ctx, void *stream) {
    if (!ctx) return fail(RLH_ERR_INVALID, "rlh_wait_stream: ctx is NULL");
    return order_streams("rlh_wait_stream", ctx, static_cast<hipStream_t>(stream), ctx->stream);
}

extern "C" int rlh_release_stream(rlh_ctx *ctx, void *stream) {
    if (!ctx) return fail(RLH_ERR_INVALID, "rlh_release_stream: ctx is NULL");
    return order_streams("rlh_release_stream", ctx, ctx->stream, static_cast<hipStream_t>(stream));
}

extern "C" int rlh_convert(rlh_tensor *dst, const rlh_tensor *src) {
    if (!dst || !src || dst->rows != src->rows || dst->cols != src->cols) return fail(RLH_ERR_INVALID, "rlh_convert: two tensors of one shape are needed");
    if (dst->dtype == RLH_I32 || src->dtype == RLH_I32) return fail(RLH_ERR_UNSUPPORTED, "rlh_convert: f16, f32, 4-bit and 8-bit tensors only");
    if (dst->dtype == src->dtype) return rlh_copy_inplace(dst, src);
    if ((dst->is_eight() && !src->is_float()) || (src->is_eight() && !dst->is_float())) return fail(RLH_ERR_UNSUPPORTED, "rlh_convert: 8 bits from and to f16 and f32 only");
    if ((dst->is_eight() || src->is_eight()) && dst->p == src->p) return fail(RLH_ERR_INVALID, "rlh_convert: tensors of 8 bits must not share memory with the other one");
    CtxLock lock(dst->ctx);
    lend(dst->ctx, {src});
    if (dst->is_eight()) {
        HIP_TRY(launch_f8_encode(eight_of(dst), src->p, src->dtype == RLH_F16, dst->rows, dst->cols, dst->ctx->stream));
        return RLH_OK;
    }
    if (src->is_eight()) {
        HIP_TRY(launch_f8_decode(dst->p, dst->dtype == RLH_F16, eight_of(src), dst->rows, dst->cols, dst->ctx->stream));
        return RLH_OK;
    }
    HIP_TRY(launch_plane_convert(plane_of(dst), plane_type(dst), plane_of(src), plane_type(src), dst->count(), dst->ctx->stream));
    return RLH_OK;
}

// What rlh_qkv_append and rlh_attn_window share: the planes, and the positions of `rows` rows.  Fills in head_dim, n and whether a position lies
// past the planes' rows.
struct RowPlan {
    int head_dim = 0, n = 0;
    bool wraps = false;
};
static int plan_rows(const char *who, const rlh_tensor *ck, const rlh_tensor *cv, int n_heads, int n_kv_heads, int max_seq_len, const int32_t *start_pos, int n_seqs,
                     int rows, RowPlan *plan) {
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads != 0) return fail(RLH_ERR_INVALID, "%s: %d heads do not share %d key and value heads evenly", who, n_heads, n_kv_heads);
    if (!start_pos || n_seqs < 1 || n_seqs > kLongMaxSeqs) return fail(RLH_ERR_INVALID, "%s: 1 to %d sequences with a position each", who, kLongMaxSeqs);
    if (!ck || !cv || max_seq_len <= 0 || ck->dtype != cv->dtype || !holds_plane(ck) || ck->rows != cv->rows || ck->cols != cv->cols ||
        (int64_t)ck->rows != (int64_t)n_seqs * n_kv_heads * max_seq_len) {
        return fail(RLH_ERR_INVALID, "%s: cache planes must be two [n_seqs * n_kv_heads * max_seq_len x head_dim] tensors of one dtype", who);
    }
    if (ck->cols != 32 && ck->cols != 64 && ck->cols != 128) return fail(RLH_ERR_UNSUPPORTED, "%s: head_dim %d (32, 64 and 128 are built)", who, ck->cols);
    if (rows % n_seqs != 0) return fail(RLH_ERR_INVALID, "%s: %d rows are not the same number for each of %d sequences", who, rows, n_seqs);
    plan->head_dim = ck->cols;
    plan->n = rows / n_seqs;
    for (int b = 0; b < n_seqs; b++) {
        const int64_t end = (int64_t)start_pos[b] + plan->n;
        if (end > kLongMaxPosition) return fail(RLH_ERR_INVALID, "%s: sequence %d: position %lld", who, b, (long long)end);
        if (end > max_seq_len) plan->wraps = true;
    }
    return RLH_OK;
}

extern "C" int rlh_qkv_append(rlh_tensor *q, const rlh_tensor *qkv, const rlh_tensor *q_norm, const rlh_tensor *k_norm, double eps, const rlh_tensor *freqs, int halves,
                              rlh_tensor *cache_k, rlh_tensor *cache_v, int n_heads, int n_kv_heads, int max_seq_len, int sinks, const int32_t *start_pos, int n_seqs) {
    if (!q || !qkv || !freqs) return fail(RLH_ERR_INVALID, "rlh_qkv_append: NULL argument");
    RowPlan plan;
    int rc = plan_rows("rlh_qkv_append", cache_k, cache_v, n_heads, n_kv_heads, max_seq_len, start_pos, n_seqs, qkv->rows, &plan);
    if (rc != RLH_OK) return rc;
    const int hd = plan.head_dim;
    if (!qkv->is_float() || q->dtype != qkv->dtype || !shaped(qkv, qkv->rows, ((int64_t)n_heads + 2 * (int64_t)n_kv_heads) * hd) || !shaped(q, qkv->rows, (int64_t)n_heads * hd)) {
        return fail(RLH_ERR_INVALID, "rlh_qkv_append: qkv must be [rows x (n_heads + 2 n_kv_heads) head_dim] and q [rows x n_heads head_dim], both f16 or both f32");
    }
    for (const rlh_tensor *w : {q_norm, k_norm})
        if (w && (w->dtype != RLH_F32 || !shaped(w, 1, hd))) return fail(RLH_ERR_INVALID, "rlh_qkv_append: norm weights must be f32 [1 x head_dim]");
    if (!(eps >= 0.0)) return fail(RLH_ERR_INVALID, "rlh_qkv_append: eps must not be negative");
    if (freqs->dtype != RLH_F32 || freqs->cols != hd) return fail(RLH_ERR_INVALID, "rlh_qkv_append: freqs must be f32 [positions x head_dim]");
    if (q->p == qkv->p || cache_k->p == cache_v->p) return fail(RLH_ERR_INVALID, "rlh_qkv_append: q and qkv, and the two planes, must not share memory");
    if (sinks < 0 || sinks >= max_seq_len) return fail(RLH_ERR_INVALID, "rlh_qkv_append: sinks %d outside 0..max_seq_len - 1", sinks);
    for (int b = 0; b < n_seqs; b++)
        if ((int64_t)start_pos[b] + plan.n > freqs->rows) return fail(RLH_ERR_STATE, "rlh_qkv_append: sequence %d reaches position %lld, freqs has %d", b, (long long)start_pos[b] + plan.n - 1, freqs->rows);
    if (plan.wraps && plan.n > max_seq_len - sinks) return fail(RLH_ERR_STATE, "rlh_qkv_append: %d rows at once in a ring of %d", plan.n, max_seq_len - sinks);
    rlh_ctx *ctx = q->ctx;
    CtxLock lock(ctx);
    lend(ctx, {qkv, freqs, cache_k, cache_v});
    for (const rlh_tensor *w : {q_norm, k_norm})
        if (w) lend(ctx, {w});
    QkvAppendParams p{};
    p.qkv = plane_of(qkv);
    p.q = plane_of(q);
    p.f16 = qkv->dtype == RLH_F16;
    p.q_norm = q_norm ? (const float *)q_norm->p : nullptr;
    p.k_norm = k_norm ? (const float *)k_norm->p : nullptr;
    p.eps = (float)eps;
    p.freqs = (const float *)freqs->p;
    p.halves = halves ? 1 : 0;
    p.cache_k = plane_of(cache_k);
    p.cache_v = plane_of(cache_v);
    p.cache = plane_type(cache_k);
    p.n_heads = n_heads;
    p.n_kv = n_kv_heads;
    p.head_dim = hd;
    p.max_seq_len = max_seq_len;
    p.sinks = sinks;
    p.n = plan.n;
    p.n_seqs = n_seqs;
    for (int b = 0; b < n_seqs; b++) p.start[b] = start_pos[b];
    HIP_TRY(launch_qkv_append(p, ctx->stream));
    return RLH_OK;
}

// Work memory of rlh_attn_window; growing it waits for the context's stream.
static hipError_t window_work_reserve(rlh_ctx *ctx, size_t floats) {
    OpScratch &o = ctx->ops;
    if (floats <= o.window_ws_floats) return hipSuccess;
    if (o.window_ws) {
        (void)hipStreamSynchronize(ctx->stream);
        (void)hipFree(o.window_ws);
        o.window_ws = nullptr;
        o.window_ws_floats = 0;
    }
    const hipError_t e = device_alloc(ctx, (void **)&o.window_ws, floats * sizeof(float));
    if (e == hipSuccess) o.window_ws_floats = floats;
    return e;
}

extern "C" int rlh_attn_window(rlh_tensor *out, const rlh_tensor *q, const rlh_tensor *cache_k, const rlh_tensor *cache_v, int n_heads, int n_kv_heads, int max_seq_len,
                               const int32_t *start_pos, int n_seqs, int window, int sinks) {
    if (!out || !q) return fail(RLH_ERR_INVALID, "rlh_attn_window: NULL argument");
    RowPlan plan;
    int rc = plan_rows("rlh_attn_window", cache_k, cache_v, n_heads, n_kv_heads, max_seq_len, start_pos, n_seqs, q->rows, &plan);
    if (rc != RLH_OK) return rc;
    const int hd = plan.head_dim;
    if (!q->is_float() || out->dtype != q->dtype || !shaped(q, q->rows, (int64_t)n_heads * hd) || !shaped(out, q->rows, (int64_t)n_heads * hd)) {
        return fail(RLH_ERR_INVALID, "rlh_attn_window: q and out must be [rows x n_heads head_dim], both f16 or both f32");
    }
    if (out->p == q->p) return fail(RLH_ERR_INVALID, "rlh_attn_window: q and out must not share memory");
    if (window < 0 || sinks < 0 || sinks >= max_seq_len) return fail(RLH_ERR_INVALID, "rlh_attn_window: window %d, sinks %d (not negative, sinks below max_seq_len)", window, sinks);
    if (plan.wraps && (window == 0 || (int64_t)sinks + window + plan.n - 1 > max_seq_len)) {
        return fail(RLH_ERR_STATE, "rlh_attn_window: positions beyond max_seq_len %d need a window, and sinks %d + window %d + rows %d - 1 within it", max_seq_len, sinks, window, plan.n);
    }
    rlh_ctx *ctx = out->ctx;
    CtxLock lock(ctx);
    lend(ctx, {q, cache_k, cache_v});
    AttnWindowParams p{};
    p.q = q->p;
    p.out = out->p;
    p.f16 = q->dtype == RLH_F16;
    p.cache_k = plane_of(cache_k);
    p.cache_v = plane_of(cache_v);
    p.cache = plane_type(cache_k);
    p.n_heads = n_heads;
    p.n_kv = n_kv_heads;
    p.head_dim = hd;
    p.max_seq_len = max_seq_len;
    p.n = plan.n;
    p.n_seqs = n_seqs;
    p.window = window;
    p.sinks = sinks;
    p.exact = ctx->tun.attn_exact;
    for (int b = 0; b < n_seqs; b++) p.start[b] = start_pos[b];
    const int cus = ctx->prop.multiProcessorCount;
    const int64_t rows = (int64_t)p.n * (n_heads / n_kv_heads), most = attn_window_most_rows(p, cus);
    if (rows > most) return fail(RLH_ERR_UNSUPPORTED, "rlh_attn_window: %lld rows on one key and value head, %lld at once (65535 sequences and key heads)", (long long)rows, (long long)most);
    HIP_TRY(window_work_reserve(ctx, attn_window_work_floats(p, cus)));
    HIP_TRY(launch_attn_window(p, cus, ctx->ops.window_ws, ctx->stream));
    return RLH_OK;
}

extern "C" int rlh_softmax_rows(rlh_tensor *probs, const rlh_tensor *logits, float temperature) {
    if (!probs || !logits || probs->dtype != RLH_F32 || !logits->is_float() || !shaped(probs, logits->rows, logits->cols)) {
        return fail(RLH_ERR_INVALID, "rlh_softmax_rows: logits f16 or f32 and probs f32 of one shape are needed");
    }
    if (!(temperature >= 0.0f) || std::isinf(temperature)) return fail(RLH_ERR_INVALID, "rlh_softmax_rows: temperature %g", (double)temperature);
    CtxLock lock(probs->ctx);
    lend(probs->ctx, {logits});
    HIP_TRY(launch_softmax_rows((float *)probs->p, logits->p, logits->dtype == RLH_F16, logits->rows, logits->cols, temperature, probs->ctx->stream));
    return RLH_OK;
}

extern "C" int rlh_verify_draft(rlh_tensor *out, const rlh_tensor *target, const rlh_tensor *draft, const rlh_tensor *drafted, const rlh_tensor *uniforms) {
    if (!out || !target || !drafted || !uniforms) return fail(RLH_ERR_INVALID, "rlh_verify_draft: NULL argument");
    const int64_t b = drafted->rows, k = drafted->cols, v = target->cols;
    if (drafted->dtype != RLH_I32 || out->dtype != RLH_I32 || !shaped(out, b, k + 2)) return fail(RLH_ERR_INVALID, "rlh_verify_draft: drafted i32 [n_seqs x k] and out i32 [n_seqs x (k + 2)] are needed");
    if (target->dtype != RLH_F32 || !shaped(target, b * (k + 1), v) || (draft && (draft->dtype != RLH_F32 || !shaped(draft, b * k, v)))) {
        return fail(RLH_ERR_INVALID, "rlh_verify_draft: target f32 [n_seqs (k + 1) x vocab] and draft f32 [n_seqs k x vocab] are needed");
    }
    if (uniforms->dtype != RLH_F32 || !shaped(uniforms, b, k + 1)) return fail(RLH_ERR_INVALID, "rlh_verify_draft: uniforms f32 [n_seqs x (k + 1)] are needed");
    CtxLock lock(out->ctx);
    lend(out->ctx, {target, drafted, uniforms});
    if (draft) lend(out->ctx, {draft});
    VerifyParams p{};
    p.target = (const float *)target->p;
    p.draft = draft ? (const float *)draft->p : nullptr;
    p.drafted = (const int32_t *)drafted->p;
    p.uniforms = (const float *)uniforms->p;
    p.out = (int32_t *)out->p;
    p.n_seqs = (int)b;
    p.k = (int)k;
    p.vocab = (int)v;
    HIP_TRY(launch_verify_draft(p, out->ctx->stream));
    return RLH_OK;
}
