// check_answers_main.cpp -- the tensor methods of rllama_hip.hpp for many answers to one prompt as a program: reads one step's inputs from a file, runs it through the
// C++ mirror and writes what comes out (tests/test_gpu_answers_mirror.py compares with the same calls from Python).
//
//   rllama_check_answers IN OUT [PARTS]
//
// IN: nine int32 (heads, key and value heads, head size, texts, prefix, cache rows of a text, vocabulary, tokens of a row, alternatives), then f32: the prompt's rows of the
// projection [prefix x (heads + 2 kv) hd], rows of the step [texts x heads hd], weights of the projection and of the output head; i32: positions of the texts, tokens.
// OUT: attention f32, the head's weights as their 8-bit buffer, logits f32, log probabilities, entropies, ids and log probabilities of the alternatives.
// PARTS: the same calls with what may be left out: attention without a prefix f32; log probabilities and entropies without alternatives; entropies, ids and log probabilities of the
// alternatives without tokens; attention times the head's weights in the rows' own type, f32, and from 8 bits, f16.
#include "rllama_hip.hpp"

#include <cstdio>
#include <cstring>
#include <fstream>
#include <iterator>

using rllama::Tensor;
using rllama::TensorDType;

static void put(std::ofstream &to, const Tensor &t, size_t bytes) {
    std::vector<char> host(bytes);
    t.to_cpu(host.data(), t.cols());
    to.write(host.data(), (std::streamsize)bytes);
}

static int run(const char *in_path, const char *out_path, const char *parts_path) {
    std::ifstream in(in_path, std::ios::binary);
    const std::vector<char> data((std::istreambuf_iterator<char>(in)), std::istreambuf_iterator<char>());
    int32_t n[9];
    if (data.size() < sizeof n) throw std::runtime_error("no input");
    std::memcpy(n, data.data(), sizeof n);
    const int heads = n[0], kv = n[1], hd = n[2], texts = n[3], prefix = n[4], cache_rows = n[5], vocab = n[6], m = n[7], top = n[8], dim = heads * hd, wide = (heads + 2 * kv) * hd;
    size_t at = sizeof n;
    auto cl = std::make_shared<rllama::OpenCL>(false, 0);
    auto next = [&](int64_t r, int64_t c, TensorDType dtype) {
        const size_t bytes = (size_t)(r * c) * 4;
        if (at + bytes > data.size()) throw std::runtime_error("input too short");
        Tensor t(cl, data.data() + at, r, c, c, dtype);
        at += bytes;
        return t;
    };
    const Tensor prompt = next(prefix, wide, TensorDType::Float32), x = next(texts, dim, TensorDType::Float32);
    const Tensor w_qkv = next(wide, dim, TensorDType::Float32).convert(TensorDType::Float8Tiles), w_head = next(vocab, dim, TensorDType::Float32).convert(TensorDType::Float8Tiles);
    std::vector<int32_t> starts((size_t)texts);
    if (at + starts.size() * 4 > data.size()) throw std::runtime_error("input too short");
    std::memcpy(starts.data(), data.data() + at, starts.size() * 4);
    at += starts.size() * 4;
    const Tensor tokens = next(texts, m, TensorDType::Int32);

    auto plane = [&](int64_t rows) { return Tensor::zeros(cl, rows, hd, TensorDType::Float16); };
    Tensor prefix_k = plane((int64_t)kv * prefix), prefix_v = plane((int64_t)kv * prefix), cache_k = plane((int64_t)texts * kv * cache_rows), cache_v = plane((int64_t)texts * kv * cache_rows);
    prompt.qkv_append(prefix_k, prefix_v, Tensor::rope_table(cl, prefix, hd), heads, kv, prefix, {0});
    const Tensor behind = Tensor::rope_table_from(cl, prefix, cache_rows, hd);
    const Tensor q = x.matrix_mul_f8(w_qkv, TensorDType::Float32).qkv_append(cache_k, cache_v, behind, heads, kv, cache_rows, starts);
    const Tensor out = q.attn_shared(prefix_k, prefix_v, prefix, cache_k, cache_v, heads, kv, cache_rows, starts);
    const Tensor logits = out.convert(TensorDType::Float8).matrix_mul_f8(w_head, TensorDType::Float32);
    const Tensor::Logprobs p = logits.token_logprobs(tokens, top, 0.7f);

    std::ofstream to(out_path, std::ios::binary);
    put(to, out, (size_t)texts * dim * 4);
    put(to, w_head, (size_t)vocab * dim + (size_t)((vocab + 127) / 128) * ((dim + 127) / 128) * 4);
    put(to, logits, (size_t)texts * vocab * 4);
    put(to, p.logprobs, (size_t)texts * m * 4);
    put(to, p.entropy, (size_t)texts * 4);
    put(to, p.top_ids, (size_t)texts * top * 4);
    put(to, p.top_logprobs, (size_t)texts * top * 4);
    to.flush();
    if (!to) return 1;
    if (!parts_path) return 0;

    const Tensor alone = q.attn_shared(cache_k, cache_v, heads, kv, cache_rows, starts);
    const Tensor::Logprobs given = logits.token_logprobs(tokens), best = logits.token_logprobs(top, 0.7f);
    if (!given.top_ids.empty() || !given.top_logprobs.empty() || !best.logprobs.empty()) throw std::runtime_error("results that were not asked for");
    const Tensor whole = out.matrix_mul_f8(w_head), narrow = out.convert(TensorDType::Float8).matrix_mul_f8(w_head);
    if (whole.dtype() != TensorDType::Float32 || narrow.dtype() != TensorDType::Float16) throw std::runtime_error("results of another type");
    std::ofstream parts(parts_path, std::ios::binary);
    put(parts, alone, (size_t)texts * dim * 4);
    put(parts, given.logprobs, (size_t)texts * m * 4);
    put(parts, given.entropy, (size_t)texts * 4);
    put(parts, best.entropy, (size_t)texts * 4);
    put(parts, best.top_ids, (size_t)texts * top * 4);
    put(parts, best.top_logprobs, (size_t)texts * top * 4);
    put(parts, whole, (size_t)texts * vocab * 4);
    put(parts, narrow, (size_t)texts * vocab * 2);
    parts.flush();
    return parts ? 0 : 1;
}

int main(int argc, char **argv) {
    if (argc != 3 && argc != 4) {
        std::fprintf(stderr, "usage: rllama_check_answers IN OUT [PARTS]\n");
        return 2;
    }
    try {
        return run(argv[1], argv[2], argc > 3 ? argv[3] : nullptr);
    } catch (const std::exception &e) {
        std::fprintf(stderr, "%s\n", e.what());
        return 1;
    }
}
