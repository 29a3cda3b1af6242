// check_tensors_main.cpp -- the tensor methods of rllama_hip.hpp for long contexts and drafted tokens as a program: reads one step's inputs from a file, runs it
// through the C++ mirror and writes what comes out (tests/test_gpu_longctx_mirror.py compares with the same calls from Python).
//
//   rllama_check_tensors IN OUT
//
// IN: nine int32 (heads, key and value heads, head size, rows, cache rows, window, sinks, vocabulary, drafted tokens k), then qkv f16, norms of queries and of keys
// f32, logits f32 [k + 1 x vocabulary], probabilities of the draft f32 [k x vocabulary], drafted ids i32 [k], variates f32 [k + 1].
// OUT: attention f16, the keys' plane as its 4-bit buffer and as f32, the result of the verification with the draft's probabilities and without.
#include "rllama_hip.hpp"

#include <cstdio>
#include <cstring>
#include <dlfcn.h>
#include <fstream>
#include <iterator>

using rllama::Tensor;
using rllama::TensorDType;

static void put(std::ofstream &to, const Tensor &t, size_t bytes) {
    std::vector<char> host(bytes);
    t.to_cpu(host.data(), t.cols());
    to.write(host.data(), (std::streamsize)bytes);
}

static int run(const char *in_path, const char *out_path) {
    std::ifstream in(in_path, std::ios::binary);
    const std::vector<char> data((std::istreambuf_iterator<char>(in)), std::istreambuf_iterator<char>());
    int32_t n[9];
    if (data.size() < sizeof n) throw std::runtime_error("no input");
    std::memcpy(n, data.data(), sizeof n);
    const int heads = n[0], kv = n[1], hd = n[2], rows = n[3], cache_rows = n[4], window = n[5], sinks = n[6], vocab = n[7], k = n[8];
    size_t at = sizeof n;
    auto cl = std::make_shared<rllama::OpenCL>(false, 0);
    auto next = [&](int64_t r, int64_t c, TensorDType dtype) {
        const size_t bytes = (size_t)(r * c) * (dtype == TensorDType::Float16 ? 2 : 4);
        if (at + bytes > data.size()) throw std::runtime_error("input too short");
        Tensor t(cl, data.data() + at, r, c, c, dtype);
        at += bytes;
        return t;
    };
    const Tensor qkv = next(rows, (int64_t)(heads + 2 * kv) * hd, TensorDType::Float16);
    const Tensor q_norm = next(1, hd, TensorDType::Float32), k_norm = next(1, hd, TensorDType::Float32);
    // the logits from device memory that is not the library's
    const auto device_malloc = reinterpret_cast<int (*)(void **, size_t)>(dlsym(RTLD_DEFAULT, "hipMalloc"));
    const auto device_copy = reinterpret_cast<int (*)(void *, const void *, size_t, int)>(dlsym(RTLD_DEFAULT, "hipMemcpy"));
    void *memory = nullptr; // (the process's until it ends)
    const size_t logit_bytes = (size_t)(k + 1) * vocab * 4;
    if (at + logit_bytes > data.size()) throw std::runtime_error("input too short");
    if (!device_malloc || !device_copy || device_malloc(&memory, logit_bytes) != 0 || device_copy(memory, data.data() + at, logit_bytes, 1 /* to the device */) != 0)
        throw std::runtime_error("no device memory");
    at += logit_bytes;
    const Tensor logits = Tensor::from_device(cl, memory, k + 1, vocab, TensorDType::Float32), draft = next(k, vocab, TensorDType::Float32);
    const Tensor drafted = next(1, k, TensorDType::Int32), uniforms = next(1, k + 1, TensorDType::Float32);

    const Tensor freqs = Tensor::rope_table(cl, rows, hd);
    Tensor cache_k = Tensor::zeros(cl, (int64_t)kv * cache_rows, hd, TensorDType::K4BitQuantization), cache_v = Tensor::zeros(cl, (int64_t)kv * cache_rows, hd, TensorDType::K4BitQuantization);
    cl->wait_stream(nullptr);
    const Tensor q = qkv.qkv_append(cache_k, cache_v, freqs, heads, kv, cache_rows, {0}, &q_norm, &k_norm, 1e-5, true, sinks);
    const Tensor out = q.attn_window(cache_k, cache_v, heads, kv, cache_rows, {0}, window, sinks);
    const Tensor probs = logits.softmax_rows(0.8f);
    const Tensor with = drafted.verify_draft(probs, &draft, uniforms), without = drafted.verify_draft(probs, nullptr, uniforms);
    cl->release_stream(nullptr);

    std::ofstream to(out_path, std::ios::binary);
    const size_t count = (size_t)kv * cache_rows * hd;
    put(to, out, (size_t)rows * heads * hd * 2);
    put(to, cache_k, count / 32 * 20);
    // a saved plane comes back as it was
    std::vector<char> saved(count / 32 * 20);
    cache_k.to_cpu(saved.data(), hd);
    put(to, Tensor(cl, saved.data(), cache_k.rows(), hd, hd, TensorDType::K4BitQuantization).convert(TensorDType::Float32), count * 4);
    put(to, with, (size_t)(k + 2) * 4);
    put(to, without, (size_t)(k + 2) * 4);
    to.flush();
    return to ? 0 : 1;
}

int main(int argc, char **argv) {
    if (argc != 3) {
        std::fprintf(stderr, "usage: rllama_check_tensors IN OUT\n");
        return 2;
    }
    try {
        return run(argv[1], argv[2]);
    } catch (const std::exception &e) {
        std::fprintf(stderr, "%s\n", e.what());
        return 1;
    }
}
